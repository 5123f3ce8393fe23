// The fp8 linear operator's kernels (irodori_op_linear_fp8): Y = R + G * act(sum_b sx[m, b] sw[n / 128, b] (X W^T)_b + b),
// (X W^T)_b the product over the b-th 128 of K of the e4m3 codes X [M, K] and W [N, K], on the matrix cores with f32 sums.
//
// A block's product starts from zero in registers of its own and joins the tile's sums by one multiply-add an element
// with sx sw in f32: the product is formed transposed (W's rows are the A operand), so a lane has one row of Y and one factor a
// block.  The 16x16x128 step takes a block at once; its 4 multiply-adds take half of its cycles and run beside others' (register
// to register, random codes: 3.1 PFLOP/s with them, 3.7 without; the 32x32x64 step 2.8 and 3.6).  The epilogue is the linear operator's.
//
// The fp8 matrix instructions align each 8 products of neighbouring codes to the largest and keep 13 bits below its exponent
// (measured; beyond the 8 their sums are f32): 1.4e-5 relative L2 for normal operands, 3.8e-5 with a few channels of 16 times the rest, far
// below the rounding of a 16-bit Y (1.7e-3 bf16, 2.1e-4 f16).  An f32 Y takes the codes as bf16, which holds them and their products exactly, at half of the rate (1e-7);
// so do few rows, which wait for W.
//
// Large tiles (128 x 256 and up, 16-bit outputs) are taken one after another by a workgroup a CU, whose loads run a slice ahead of its
// products across them.  Measured a call, host side included (the operator's floor at the library's 2489 TFLOP/s, or a copy's 5.1 TB/s):
//   4 x 7360 x 1280                      7.2 us [1.9]   the call; W at 1.8 TB/s in 5.1 us of kernel
//   253 x 1280 x 1000 f16, gelu          7.6 [0.4]      the call; a chain of two slices and the epilogue
//   1500 x 1024 x 2816 -> f32, gate, residual  16.4 [3.8]  bf16 products (7.4 at the library's rate): 11 slices a tile of which the codes'
//                                        widening takes as many cycles as the products
//   24000 x 5632 x 1024                  152-160 [111]  by machine; on one 148, and 126 without the epilogue: its stores 22 (53 at a copy's rate, the
//                                        rest under products); 8192^3 takes 482-513 where the library's product without blocks' scales takes 442
#include <type_traits>

#include "attn_util.hpp"
#include "fp8_block.hpp"
#include "kernels.hpp"
#include "linear_fp8.hpp"
#include "linear_tile.hpp"

namespace irodori {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
// A uniform value, by the scalar cache.
typedef const __attribute__((address_space(4))) float* uniform_ptr;
__device__ __forceinline__ uniform_ptr uniform(const float* p) { return (uniform_ptr)(uintptr_t)p; }

// The 32 codes a lane (row r, quarter g = lane / 16) supplies of a block: K bytes 16 g .. + 15 and 64 more on.  An LDS row has a
// block, or several (RB bytes); b is the block in it.
typedef const __attribute__((address_space(3))) unsigned char* lds_ptr;
__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(uintptr_t)(lds_ptr)p; }
struct Pieces {
    unsigned lo, hi;  // the LDS addresses of the two
};
template <int RB>
__device__ __forceinline__ Pieces pieces_of(unsigned row, int r, int b, int g) {
    return {row + (lswz<RB>(r, 8 * b + g) << 4), row + (lswz<RB>(r, 8 * b + 4 + g) << 4)};
}
// `further`: a constant number of bytes.
__device__ __forceinline__ i32x8 read_codes(const Pieces& p, int further) {
    typedef const __attribute__((address_space(3))) u32x4* piece_ptr;
    const u32x4 lo = *(piece_ptr)((lds_ptr)(uintptr_t)p.lo + further), hi = *(piece_ptr)((lds_ptr)(uintptr_t)p.hi + further);
    i32x8 f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        f[e] = lo[e];
        f[4 + e] = hi[e];
    }
    return f;
}
// Codes 8 q .. 8 q + 7 of a lane's 32 as bf16, exactly.
__device__ __forceinline__ bf16x8 widen(const i32x8& v, int q) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * q + i], 1.f, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * q + i], 1.f, true);
        r[4 * i] = lo[0];
        r[4 * i + 1] = lo[1];
        r[4 * i + 2] = hi[0];
        r[4 * i + 3] = hi[1];
    }
    return r;
}
// A block's product: of the codes, or of their bf16 values.
template <bool EXACT>
struct Operand {
    i32x8 v;
    __device__ __forceinline__ void set(const i32x8& c) { v = c; }
};
template <>
struct Operand<true> {
    bf16x8 v[4];
    __device__ __forceinline__ void set(const i32x8& c) {
#pragma unroll
        for (int q = 0; q < 4; q++) v[q] = widen(c, q);
    }
};
__device__ __forceinline__ f32x4 product(const Operand<false>& a, const Operand<false>& b) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, zero, 0, 0, 0, 0, 0, 0);  // (the form without block scales)
}
__device__ __forceinline__ f32x4 product(const Operand<true>& a, const Operand<true>& b) {
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; q++) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], p, 0, 0, 0);
    return p;
}
__device__ __forceinline__ bool any_lane(bool b) { return __builtin_amdgcn_ballot_w64(b) != 0; }
__device__ __forceinline__ bool normal(float f) { return __builtin_amdgcn_classf(f, 0x108); }
// Scales far apart: their product f is no normal f32 number, though both are numbers other than 0.  A block's sum p (0 or from 2^-18 to 2^25 in
// magnitude) times them is (p up) rest then, with `up` 2^64 or 2^-64 and the rest a normal number; what passes an end of f32's range so
// passes it by itself.  The tiles' loop takes f as it is: one that is subnormal or 0 is off by 2^-150, its term by less than 2^-125; one that
// is infinite is seen to after it.
__device__ __forceinline__ bool far_apart(float sx, float sw) {
    auto number = [](float v) { return __builtin_amdgcn_classf(v, 0x198); };  // normal or subnormal
    return !normal(sx * sw) && number(sx) && number(sw);
}
struct Factor {
    float up, rest;
    __device__ __forceinline__ Factor(float sx, float sw) {
        const float f = sx * sw, by = fabsf(f) < 1.f ? 0x1p32f : 0x1p-32f;
        const bool apart = far_apart(sx, sw);
        up = !apart ? 1.f : fabsf(f) < 1.f ? 0x1p-64f : 0x1p64f;
        rest = !apart ? f : fminf(fmaxf((sx * by) * (sw * by), -3.402823466e38f), 3.402823466e38f);
    }
};
// 16 bytes a lane from a buffer window to LDS at `to` (the same in every lane) and 16 times the lane.  By hand, since behind the
// builtin the compiler lets every LDS read wait for all loads on their way; the waits are wait_vm's.  (5 wait states: what a window in
// registers that the vector unit has just written takes; the compiler does not look for hazards in here.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is the compiler's, which has to know that it changes)
typedef unsigned Window __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Window make_window(const void* base, unsigned bytes) {
    const uint64_t p = (uint64_t)(uintptr_t)base;
    return Window{(unsigned)p, (unsigned)(p >> 32), bytes, 0x00020000u};
}
__device__ __forceinline__ void load_to_lds(Window w, unsigned offset, unsigned to) {
    const int at = __builtin_amdgcn_readfirstlane((int)to);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(offset), "s"(w)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
// The dword of codes that begins at k without those past K.
__device__ __forceinline__ int cut_dword(int v, int k, int K) {
    const int left = K - k;
    return left >= 4 ? v : left <= 0 ? 0 : v & ((1 << 8 * left) - 1);
}
// The 16 codes from lo on and the 16 from hi on of a row at p, those past K zero (WHOLE: there are none).
template <bool WHOLE>
__device__ __forceinline__ i32x8 load_codes(const unsigned char* p, int lo, int hi, int K) {
    typedef unsigned U4 __attribute__((ext_vector_type(4), aligned(1)));
    i32x8 f;
    if (WHOLE || hi + 16 <= K) {
        const U4 l = *reinterpret_cast<const U4*>(p + lo), h = *reinterpret_cast<const U4*>(p + hi);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f[e] = l[e];
            f[4 + e] = h[e];
        }
        return f;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        unsigned v = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = (e < 4 ? lo : hi - 16) + 4 * e + i;
            if (k < K) v |= (unsigned)p[k] << (8 * i);
        }
        f[e] = v;
    }
    return f;
}
// W's row of a wave's 16 FN that operand row r of its block i takes, so that a lane ends with 4 FN neighbouring columns of one row of Y,
// and the operand row of W's row w.
template <int FN>
__device__ __forceinline__ int w_row16(int i, int r) {
    return 4 * FN * (r >> 2) + 4 * i + (r & 3);
}
template <int FN>
__device__ __forceinline__ int operand_row16(int w) {
    return 4 * (w / (4 * FN) % 4) + (w & 3);
}

// A tile of BM rows and BN columns of Y per workgroup of WM x WN x WK wavefronts.  K advances in slices of WK blocks of 128
// codes, one for each of the WK, which are summed through LDS at the end.  ASYNC: slices move HBM -> LDS by
// buffer_load_dwordx4 ... lds, which take dword-aligned rows; a piece that straddles K's end is cut
// in the last slice.  Otherwise through registers.  The scales of X come along every fourth block.
template <typename TO, int BM, int BN, int WM, int WN, int WK, int STAGES, bool ASYNC, bool AHEAD, int EU>
__global__ __launch_bounds__(64 * WM * WN * WK) __attribute__((amdgpu_waves_per_eu(EU, EU))) void linear_fp8_kernel(LinearFp8Args args) {
    const LinearArgs& a = args.l;
    constexpr bool EXACT = sizeof(TO) == 4;
    constexpr int NW = WM * WN * WK, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
    constexpr int RB = 128 * WK, ROWS = BM + BN, STAGE = ROWS * RB, RC = RB / 16;
    constexpr int RPI = 64 / RC, LPW = ROWS / RPI / NW, LW = BN / RPI / NW;  // rows a load instruction fills; a wave's per slice, W's of them
    constexpr int PER = 4 / WK, SLOTS = WK == 4 ? STAGES : 2;  // slices that share a load of scales, loads held
    constexpr int SROWS = (BM + 63) / 64 * 64;
    constexpr int C = 4 * FN;  // neighbouring columns of Y a lane ends with
    static_assert(LPW * RPI * NW == ROWS && LW * RPI * NW == BN && NW * 64 >= SROWS && 128 % TN == 0, "slices split over the waves");
    static_assert(WK == 1 || (WK - 1) * BM * BN * 4 <= STAGES * STAGE, "the k groups' sums fit the ring");
    static_assert(STAGES <= 3, "a load of scales is replaced when the slices of the one before it are all read");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[STAGES * STAGE];
    __shared__ __attribute__((aligned(1024))) float xscale[SLOTS][SROWS][4], wscale[SLOTS][64][4];
    __shared__ __attribute__((aligned(1024))) u32x4 turned[AHEAD ? 1 : NW][128];  // 16 rows of Y on their way out

    const int lane = threadIdx.x & 63, fr = lane & 15, fg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wk = wave / (WM * WN), wmn = wave % (WM * WN), wm = wmn / WN, wn = wmn % WN;
    const int nk = (args.blocks + WK - 1) / WK;
    // Groups of 8 row tiles sweep the column tiles.  An XCD takes a run of neighbouring tiles: each of its workgroups one, or, where the
    // launch has fewer workgroups than tiles, every stride-th of the run.
    const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN;
    struct Tile {
        int m0, n0, rows_m, rows_n;
    };
    auto locate = [&](int pid) __attribute__((always_inline)) {
        const int group = pid / (8 * tiles_n), first = group * 8;
        const int gm = tiles_m - first < 8 ? tiles_m - first : 8, local = pid - group * 8 * tiles_n;
        const int m0 = (first + local % gm) * BM, n0 = (local / gm) * BN;
        return Tile{m0, n0, a.M - m0 < BM ? a.M - m0 : BM, a.N - n0 < BN ? a.N - n0 : BN};
    };
    int pid, last = 0, stride = 1;  // this workgroup's tiles: pid, pid + stride, .. below last
    if (AHEAD || gridDim.x % 8) {
        pid = xcd_remap(blockIdx.x, gridDim.x);
    } else {
        const int64_t tiles = (int64_t)tiles_m * tiles_n, xcd = blockIdx.x % 8;
        stride = gridDim.x / 8;
        pid = (int)(tiles * xcd / 8) + blockIdx.x / 8;
        last = (int)(tiles * (xcd + 1) / 8);
        if (pid >= last) return;
    }
    int now = pid;  // the tile that is multiplied; pid the one that is loaded
    Tile tile = locate(now);

    // Load instruction i of this wave fills stage rows RPI (i NW + wave) .. (the first LW instructions W rows, the others X rows):
    // lane -> row lane / RC, physical chunk lane % RC, which holds the row's chunk `chunk`.
    auto chunk = [&](int i) {
        const int r = (i * NW + wave) * RPI + lane / RC;
        return lswz<RB>(i < LW ? operand_row16<FN>(r) : r, lane % RC);
    };
    [[maybe_unused]] Window rX, rW, rXS, rWS;
    [[maybe_unused]] auto look_at = [&](const Tile& t) __attribute__((always_inline)) {  // the windows of a tile's operands
        const int wblocks = (t.n0 % kBlock + t.rows_n + kBlock - 1) / kBlock;
        // Windows end with the last row's last whole dword (its other bytes are in the same memory word).
        rX = make_window(static_cast<const unsigned char*>(a.x) + (int64_t)t.m0 * a.ldx, ((unsigned)((int64_t)(t.rows_m - 1) * a.ldx + a.K) + 3) & ~3u);
        rW = make_window(static_cast<const unsigned char*>(a.w) + (int64_t)t.n0 * a.ldw, ((unsigned)((int64_t)(t.rows_n - 1) * a.ldw + a.K) + 3) & ~3u);
        rXS = make_window(args.xs + (int64_t)t.m0 * args.ldxs, (unsigned)((int64_t)(t.rows_m - 1) * args.ldxs + args.blocks) * 4u);
        rWS = make_window(args.ws + (int64_t)(t.n0 / kBlock) * args.ldws, (unsigned)((int64_t)(wblocks - 1) * args.ldws + args.blocks) * 4u);
    };
    if constexpr (ASYNC) look_at(tile);
    // Where load instruction i of slice kt reads, whole in the part that is checked against the window.  Rows past the last lie behind it
    // and read as zero, as do pieces of its last row past K (with rows closer than K apart they hold codes, which none of Y's sees).
    constexpr int STEP = NW * RPI;  // rows from one instruction of a wave to the next
    constexpr bool SAME = STEP % (16 * FN) == 0;  // a lane's chunk is the same in all of them
    [[maybe_unused]] unsigned woff[SAME ? 1 : LW], xoff[SAME ? 1 : LPW - LW];
    if constexpr (ASYNC) {
#pragma unroll
        for (int i = 0; i < (SAME ? 1 : LW); i++) woff[i] = (wave * RPI + lane / RC) * (unsigned)a.ldw + 16u * chunk(i);
#pragma unroll
        for (int i = 0; i < (SAME ? 1 : LPW - LW); i++) xoff[i] = (wave * RPI + lane / RC) * (unsigned)a.ldx + 16u * chunk(LW + i);
    }
    [[maybe_unused]] auto offset = [&](int kt, int i) __attribute__((always_inline)) {
        unsigned step = (i < LW ? i * (unsigned)a.ldw : (i - LW) * (unsigned)a.ldx) * STEP + kt * RB;
        if constexpr (!AHEAD) asm volatile("" : "+s"(step));  // (added where it is used: registers are few)
        return (i < LW ? woff[SAME ? 0 : i] : xoff[SAME ? 0 : i - LW]) + step;
    };
    [[maybe_unused]] const unsigned xsoff = (64 * wave + lane) * (unsigned)args.ldxs * 4u, wsoff = lane * (unsigned)args.ldws * 4u;
    // Slice kt into its ring slot; without ASYNC the slice that `stash` holds, and the next into it.
    [[maybe_unused]] u32x4 stash[LPW];
    [[maybe_unused]] f32x4 xstash, wstash;
    [[maybe_unused]] auto load_stash = [&](int kt) __attribute__((always_inline)) {
        const unsigned char* X = static_cast<const unsigned char*>(a.x) + (int64_t)tile.m0 * a.ldx;
        const unsigned char* W = static_cast<const unsigned char*>(a.w) + (int64_t)tile.n0 * a.ldw;
        const float *XS = args.xs + (int64_t)tile.m0 * args.ldxs, *WS = args.ws + (int64_t)(tile.n0 / kBlock) * args.ldws;
        const int wblocks = (tile.n0 % kBlock + tile.rows_n + kBlock - 1) / kBlock;
        typedef unsigned U4 __attribute__((ext_vector_type(4), aligned(1)));
#pragma unroll
        for (int i = 0; i < LPW; i++) {
            const int r = (i * NW + wave) * RPI + lane / RC - (i < LW ? 0 : BN), k = kt * RB + chunk(i) * 16;
            u32x4 v = {0u, 0u, 0u, 0u};
            if (r < (i < LW ? tile.rows_n : tile.rows_m) && k < a.K) {
                const unsigned char* src = (i < LW ? W + r * a.ldw : X + r * a.ldx) + k;
                if (k + 16 <= a.K) {
                    v = *reinterpret_cast<const U4*>(src);
                } else {
#pragma unroll
                    for (int e = 0; e < 15; e++)
                        if (k + e < a.K) v[e / 4] |= (unsigned)src[e] << (8 * (e & 3));
                }
            }
            stash[i] = v;
        }
        if (kt % PER == 0) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool there = kt * WK + e < args.blocks;
                xstash[e] = there && (int)threadIdx.x < tile.rows_m ? XS[threadIdx.x * args.ldxs + kt * WK + e] : 0.f;
                wstash[e] = there && lane < wblocks ? WS[lane * args.ldws + kt * WK + e] : 0.f;
            }
        }
    };
    // (ring, scales: the numbers of the slices and of the loads of scales so far.)
    auto issue = [&](int kt, int ring, int scales) __attribute__((always_inline)) {
        if (kt % PER == 0) {
            const int slot = scales % SLOTS;
            if constexpr (ASYNC) {
                if (wave < SROWS / 64) load_to_lds(rXS, xsoff + kt * WK * 4u, lds_address(xscale) + (slot * SROWS + 64 * wave) * 16);
                if (wave == NW - 1) load_to_lds(rWS, wsoff + kt * WK * 4u, lds_address(wscale) + slot * 64 * 16);
            } else {
                if (wave < SROWS / 64) *reinterpret_cast<f32x4*>(&xscale[slot][64 * wave + lane][0]) = xstash;
                if (wave == NW - 1) *reinterpret_cast<f32x4*>(&wscale[slot][lane][0]) = wstash;
            }
        }
        const int dst = ring % STAGES * STAGE + wave * 1024;
        if constexpr (ASYNC) {
#pragma unroll
            for (int i = 0; i < LPW; i++) load_to_lds(i < LW ? rW : rX, offset(kt, i), lds_address(smem) + dst + i * NW * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < LPW; i++) *reinterpret_cast<u32x4*>(smem + dst + i * NW * 1024 + 16 * lane) = stash[i];
            if (kt + 1 < nk) load_stash(kt + 1);
        }
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int j = 0; j < FM; j++)
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[j][i][e] = 0.f;

    // Where K ends inside the last slice, what lies past it (the next rows' codes) becomes zero.
    [[maybe_unused]] auto cut_tail = [&](int kt, int ring) __attribute__((always_inline)) {
        int t = threadIdx.x, left = a.K - kt * RB;
        asm volatile("" : "+v"(t), "+s"(left));  // (formed here, not kept in registers through the loop)
        for (int p = t; p < ROWS * RC; p += 64 * NW) {
            const int r = p / RC, k = 16 * (p % RC);
            if (k + 16 <= left) continue;
            u32x4* piece = reinterpret_cast<u32x4*>(smem + ring % STAGES * STAGE + r * RB + (lswz<RB>(r < BN ? operand_row16<FN>(r) : r, p % RC) << 4));
            u32x4 v = *piece;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = cut_dword(v[e], k + 4 * e, left);
            *piece = v;
        }
        wait_lds();
        raw_barrier();
    };
    // Slice kt is there for every wave, and every wave has read the ones before it: of the later slices that were issued, A at most may
    // be on their way, and the stores of a tile that were issued after its loads (the counter keeps their order).
    [[maybe_unused]] int stores = 0;
    auto arrive = [&](int kt, int ring, auto ahead) __attribute__((always_inline)) {
        constexpr int A = decltype(ahead)::value;
        if constexpr (!AHEAD) {
            if (stores) wait_vm<2 * FM>();
            else wait_vm<0>();
            stores = 0;
        } else if constexpr (ASYNC) {
            wait_slices<A, LPW>(nk - 1 - kt < A ? nk - 1 - kt : A);
        }
        wait_lds();
        raw_barrier();
        if constexpr (ASYNC) {
            if (kt == nk - 1 && a.K % RB) cut_tail(kt, ring);
        }
    };
    // Where a lane's fragments lie in a slot: of W's block 0 and X's block 0, the others a constant further.
    const Pieces w_at = pieces_of<RB>(lds_address(smem) + (wn * TN + w_row16<FN>(0, fr)) * RB, fr, wk, fg);
    const Pieces x_at = pieces_of<RB>(lds_address(smem) + (BN + wm * TM + fr) * RB, fr, wk, fg);
    const unsigned xs_at = lds_address(xscale) + (wm * TM + fr) * 16, ws_at = lds_address(wscale) + wn * TN / kBlock * 16;  // (a wave's columns share a scale)
    struct Place {  // of a slice
        Pieces w, x;
        unsigned xs, ws;
        bool there;  // the wave's block is within K (a slice of several may end past it)
    };
    auto place = [&](int kt, int ring, int scales) __attribute__((always_inline)) {
        const unsigned slot = ring % STAGES * STAGE, from = scales % SLOTS, b = (kt * WK + wk) % 4 * 4;
        Place p{{w_at.lo + slot, w_at.hi + slot}, {x_at.lo + slot, x_at.hi + slot}, xs_at + from * (SROWS * 16) + b, ws_at + from * 1024 + b,
                WK == 1 || kt * WK + wk < args.blocks};
        asm volatile("" : "+v"(p.w.lo), "+v"(p.w.hi), "+v"(p.x.lo), "+v"(p.x.hi), "+v"(p.xs), "+v"(p.ws));  // (each read a constant further)
        return p;
    };
    auto read_w = [&](const Place& p, int i) __attribute__((always_inline)) { return read_codes(p.w, 4 * i * RB); };
    auto read_x = [&](const Place& p, int j) __attribute__((always_inline)) { return read_codes(p.x, 16 * j * RB); };
    // The scales of rows 16 j + fr and of the wave's columns; past K both 0 (what is read there is anything).
    auto read_scales = [&](const Place& p, int j, float& x, float& w) __attribute__((always_inline)) {
        typedef const __attribute__((address_space(3))) float* float_ptr;
        x = *(float_ptr)((lds_ptr)(uintptr_t)p.xs + 16 * 16 * j);
        w = *(float_ptr)((lds_ptr)(uintptr_t)p.ws);
        if (WK > 1) x = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & (p.there ? ~0u : 0u));
        if (WK > 1) w = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, w) & (p.there ? ~0u : 0u));
    };
    // A product's sums are joined two products later, under their cycles (the last two of a slice by the next one).
    f32x4 pending[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    float pending_f[2] = {0.f, 0.f};
    constexpr int PRODUCTS = FM * FN;
    static_assert(PRODUCTS % 2 == 0, "the pending two");
    auto join = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) acc[t / FN][t % FN][e] = fmaf(pending[t & 1][e], pending_f[t & 1], acc[t / FN][t % FN][e]);
        asm volatile("" : "+v"(acc[t / FN][t % FN]));  // here, not where the compiler would gather them
    };
    auto multiply = [&](const Operand<EXACT>& w, const Operand<EXACT>& x, float f, int t) __attribute__((always_inline)) {
        const f32x4 p = product(w, x);
        if constexpr (!EXACT) __builtin_amdgcn_sched_barrier(0);
        join((t + PRODUCTS - 2) % PRODUCTS);
        pending[t & 1] = p;
        pending_f[t & 1] = f;
        if constexpr (!EXACT) __builtin_amdgcn_sched_barrier(0);
    };
    // Two ways through a slice.  AHEAD: the fragments of the next one are read under this one's products, from two sets, and the slot
    // that every wave has read is filled again before the products: STAGES slices of lookahead.  Otherwise, where two sets are too
    // many registers, W's fragments have two sets and X's come one block of 16 rows ahead; the slot is filled again, and the next slice's first
    // fragments are read, under the products of the last 16 rows.
    Operand<EXACT> w[AHEAD ? 1 : 2][FN], x[2];
    [[maybe_unused]] i32x8 cw[2][AHEAD ? FN : 1], cx[2][AHEAD ? FM : 1];
    float sx[2][AHEAD ? FM : 1], sw[2];
    Place at;
    [[maybe_unused]] auto read_slice = [&](int kt, auto set) __attribute__((always_inline)) {
        at = place(kt, kt, kt / PER);
#pragma unroll
        for (int i = 0; i < FN; i++) cw[set][i] = read_w(at, i);
#pragma unroll
        for (int j = 0; j < FM; j++) {
            cx[set][j] = read_x(at, j);
            read_scales(at, j, sx[set][j], sw[set]);
        }
    };
    // (After the last slice the reads are of whatever the slot holds, which no product takes: no branch around registers.)
    [[maybe_unused]] auto slice_ahead = [&](int kt, auto cur) __attribute__((always_inline)) {
        if (kt + 1 < nk) arrive(kt + 1, kt + 1, std::integral_constant<int, STAGES - 2>{});
        read_slice(kt + 1, std::integral_constant<int, 1 - decltype(cur)::value>{});
        if (kt + STAGES < nk) issue(kt + STAGES, kt + STAGES, (kt + STAGES) / PER);
#pragma unroll
        for (int i = 0; i < FN; i++) w[0][i].set(cw[cur][i]);
#pragma unroll
        for (int j = 0; j < FM; j++) {
            x[j & 1].set(cx[cur][j]);
            const float f = sx[cur][j] * sw[cur];
#pragma unroll
            for (int i = 0; i < FN; i++) multiply(w[0][i], x[j & 1], f, j * FN + i);
        }
    };
    [[maybe_unused]] auto next_x = [&](int j) __attribute__((always_inline)) {
        x[j & 1].set(read_x(at, j));
        read_scales(at, j, sx[j & 1][0], sw[j & 1]);
    };
    // The slices of the tiles one after the other, as the loads are issued and as they are multiplied: slice kt of a tile is the ring-th.
    struct Course {
        int kt = 0, ring = 0, scales = 0;
        __device__ __forceinline__ bool next(int nk) {  // true: a tile is done
            ring++;
            const bool done = ++kt == nk;
            if (done) kt = 0;
            if (kt % PER == 0) scales++;
            return done;
        }
    };
    Course loads, products;
    bool more = true;  // tiles to load from
    [[maybe_unused]] auto issue_next = [&]() __attribute__((always_inline)) {
        if (!more) return;
        issue(loads.kt, loads.ring, loads.scales);
        if (loads.next(nk)) {
            pid += stride;
            more = pid < last;
            if (more) look_at(locate(pid));
        }
    };
    [[maybe_unused]] auto first_fragments = [&](auto set) __attribute__((always_inline)) {
        at = place(products.kt, products.ring, products.scales);
        next_x(0);
#pragma unroll
        for (int i = 0; i < FN; i++) w[set][i].set(read_w(at, i));
    };
    [[maybe_unused]] auto slice_held = [&](auto cur) __attribute__((always_inline)) {
        static_assert(AHEAD || (ASYNC && FM % 2 == 0 && STAGES == 2 && WK == 1), "the next slice's first rows take the other set; one slice on its way");
#pragma unroll
        for (int j = 0; j < FM; j++) {
            const float f = sx[j & 1][0] * sw[j & 1];
            if (j + 1 < FM) {
                next_x(j + 1);
            } else {
                products.next(nk);
                arrive(products.kt, products.ring, std::integral_constant<int, 0>{});
                issue_next();
                first_fragments(std::integral_constant<int, 1 - decltype(cur)::value>{});
            }
#pragma unroll
            for (int i = 0; i < FN; i++) multiply(w[cur][i], x[j & 1], f, j * FN + i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr std::integral_constant<int, 0> zero;
    constexpr std::integral_constant<int, 1> one;
    if constexpr (!ASYNC) load_stash(0);
    if constexpr (AHEAD) {
#pragma unroll
        for (int s = 0; s < STAGES; s++)
            if (s < nk) issue(s, s, s / PER);
        arrive(0, 0, std::integral_constant<int, STAGES - 1>{});
        read_slice(0, zero);
    } else {
        issue_next();
        arrive(0, 0, std::integral_constant<int, 0>{});
        issue_next();
        first_fragments(zero);
    }
    auto slice = [&](int kt, auto cur) __attribute__((always_inline)) {
        if constexpr (AHEAD) slice_ahead(kt, cur);
        else slice_held(cur);
    };
    auto all_slices = [&]() __attribute__((always_inline)) {
        int kt = 0;
        for (; kt + 1 < nk; kt += 2) {
            slice(kt, zero);
            slice(kt + 1, one);
        }
        if (kt < nk) {
            slice(kt, zero);
            if constexpr (!AHEAD) {
#pragma unroll
                for (int i = 0; i < FN; i++) w[0][i] = w[1][i];  // the next tile's
            }
        }
        join(PRODUCTS - 2);
        join(PRODUCTS - 1);
    };
    // Lane (fr, fg) has of row m0 + wm TM + 16 j + fr the columns from n0 + wn TN + C fg on.
    constexpr int E = kPiece<TO>, Q = kLanes<TO, C>;
    static_assert(Q * E == C, "one exchange a row");
    typedef TO OE __attribute__((ext_vector_type(E), aligned(sizeof(TO))));
    // AHEAD: what follows the products is done for all of a wave's rows at once, step by step: every load of a step is on its way before the
    // first is used, and none waits behind a store (1500 x 1024 x 2816 into f32 with gate and residual 16.4 against 17.4 us).
    [[maybe_unused]] auto epilogue = [&](auto whole) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int n = tile.n0 + wn * TN + C * fg, left = WHOLE ? C : a.N - n, t = lane & (Q - 1);
        float bias[C];
        if (a.bias && left > 0) load_cols(a.bias + n, left, bias);
        const int m = tile.m0 + wm * TM + fr;
        u32x4 r[FM][Q];
        if (a.residual) {
#pragma unroll
            for (int j = 0; j < FM; j++) load_pieces<TO, WHOLE>(a, m + 16 * j - t, n + t * E, r[j]);
        }
        float v[FM * C];
#pragma unroll
        for (int e = 0; e < FM * C; e++) v[e] = acc[e / C][e % C / 4][e % 4];
        if (left > 0) {
            if (a.bias) {
#pragma unroll
                for (int e = 0; e < FM * C; e++) v[e] += bias[e % C];
            }
            activate<TO>(v, a.act);
            if (a.gate) {
                float f[FM][C];
#pragma unroll
                for (int j = 0; j < FM; j++) {
                    const int row = m + 16 * j < a.M ? m + 16 * j : a.M - 1;
                    load_cols(a.gate + (int64_t)(row / a.gate_rows) * a.N + n, left, f[j]);
                }
#pragma unroll
                for (int e = 0; e < FM * C; e++) v[e] *= f[e / C][e % C];
            }
        }
        if (a.residual) {
#pragma unroll
            for (int j = 0; j < FM; j++) {
                exchange(r[j], lane);
#pragma unroll
                for (int s = 0; s < Q; s++) {
                    const OE o = __builtin_bit_cast(OE, r[j][s]);
#pragma unroll
                    for (int e = 0; e < E; e++) v[j * C + s * E + e] += static_cast<float>(o[e]);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < FM * C; e++) acc[e / C][e % C / 4][e % 4] = v[e];
    };
    // Pieces of 16 bytes exchanged among neighbouring lanes, a row each, and stored.
    [[maybe_unused]] auto store_rows = [&](auto whole) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int t = lane & (Q - 1), n = tile.n0 + wn * TN + C * fg + t * E, m = tile.m0 + wm * TM + fr - t;
#pragma unroll
        for (int j = 0; j < FM; j++) {
            u32x4 p[Q];
#pragma unroll
            for (int s = 0; s < Q; s++) {
                OE o;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = static_cast<TO>(acc[j][(s * E + e) / 4][e % 4]);
                p[s] = __builtin_bit_cast(u32x4, o);
            }
            exchange(p, lane);
#pragma unroll
            for (int s = 0; s < Q; s++) {
                if (m + 16 * j + s >= a.M || (!WHOLE && n >= a.N)) continue;
                TO* y = static_cast<TO*>(a.y) + (int64_t)(m + 16 * j + s) * a.ldy + n;
                const OE o = __builtin_bit_cast(OE, p[s]);
                if (WHOLE || n + E <= a.N) {
                    *reinterpret_cast<OE*>(y) = o;
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if (n + e < a.N) y[e] = o[e];
                }
            }
        }
    };
    // A tile inside Y (16-bit outputs): a wave turns 16 rows of 64 columns in LDS, so that 8 neighbouring lanes store a row's 128 bytes.
    // The wave's LDS operations keep their order, so nothing waits but the stores; addresses are a uniform one and a lane's offset.
    [[maybe_unused]] auto finish_inner = [&](auto plain, auto past) __attribute__((always_inline)) {
        static_assert(AHEAD || (C == 16 && E == 8), "16 columns a lane, in two pieces");
        u32x4* stage = turned[wave];
        auto at = [&](int row, int c) __attribute__((always_inline)) { return row * 8 + (c ^ (row >> 1 & 7)); };  // piece c of a row
        const int n = tile.n0 + wn * TN, row = lane >> 3;
        const unsigned out = (row * (unsigned)a.ldy + (lane & 7) * E) * (unsigned)sizeof(TO);
#pragma unroll
        for (int j = 0; j < FM; j++) {
            const int m = tile.m0 + wm * TM + 16 * j;
            float v[C];
#pragma unroll
            for (int e = 0; e < C; e++) v[e] = acc[j][e / 4][e % 4];
            if constexpr (!decltype(plain)::value) {
                if (a.bias) {
                    float f[C];
                    load_cols(a.bias + n + C * fg, C, f);
#pragma unroll
                    for (int e = 0; e < C; e++) v[e] += f[e];
                }
                activate<TO>(v, a.act);
                if (a.gate) {
                    float f[C];
                    load_cols(a.gate + (int64_t)((m + fr) / a.gate_rows) * a.N + n + C * fg, C, f);
#pragma unroll
                    for (int e = 0; e < C; e++) v[e] *= f[e];
                }
                if (a.residual) {
                    u32x4 p[Q];
                    const int t = lane & (Q - 1);
                    load_pieces<TO, true>(a, m + fr - t, n + C * fg + t * E, p);
                    exchange(p, lane);
#pragma unroll
                    for (int s = 0; s < Q; s++) {
                        const OE o = __builtin_bit_cast(OE, p[s]);
#pragma unroll
                        for (int e = 0; e < E; e++) v[s * E + e] += static_cast<float>(o[e]);
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < 2; s++) {
                OE o;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = static_cast<TO>(v[s * E + e]);
                stage[at(fr, 2 * fg + s)] = __builtin_bit_cast(u32x4, o);
            }
            char* y = static_cast<char*>(a.y) + ((int64_t)m * a.ldy + n) * (int64_t)sizeof(TO);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                OE* to = reinterpret_cast<OE*>(y + (int64_t)(8 * s) * a.ldy * (int64_t)sizeof(TO) + out);
                const OE o = __builtin_bit_cast(OE, stage[at(8 * s + row, lane & 7)]);
                if constexpr (decltype(past)::value) {
                    __builtin_nontemporal_store(o, to);
                    asm volatile("");  // (else the compiler takes this code and the other's for the same)
                } else {
                    *to = o;
                }
            }
        }
    };
    // An infinite product of a row's and the wave's columns' scales makes all of the row's sums infinite or NaN.  A wave that has such sums looks for
    // one, and forms its part of the tile once more where there is one, from memory.
    auto lost = [&]() __attribute__((always_inline)) {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < FM; j++) odd |= !__builtin_amdgcn_classf(acc[j][0][0], 0x1f8);  // not finite
        const int first_m = tile.m0 + wm * TM, first_n = tile.n0 + wn * TN;
        if (__builtin_expect(!any_lane(odd), true) || first_n >= a.N) return false;
        const float* ws = args.ws + (int64_t)(first_n / kBlock) * args.ldws;
#pragma unroll 1
        for (int b = 0; b < args.blocks; b++) {
            const float sw = ws[b];
            bool far = false;
#pragma unroll 1
            for (int r = lane; r < TM && first_m + r < a.M; r += 64) {
                const float sx = args.xs[(first_m + r) * args.ldxs + b];
                far |= far_apart(sx, sw) && fabsf(sx * sw) > 1.f;
            }
            if (any_lane(far)) return true;
        }
        return false;
    };
    // 16 x 16 at a time, block by block and group by group of them as above, each with a factor of two parts (rows outside the operands are
    // the last ones').
    auto once_more = [&]() __attribute__((always_inline)) {
        const int first_m = tile.m0 + wm * TM, first_n = tile.n0 + wn * TN;
        const float* ws = args.ws + (int64_t)(first_n / kBlock) * args.ldws;
#pragma unroll 1
        for (int t = 0; t < PRODUCTS; t++) {
            const int row = first_m + 16 * (t / FN) + fr, m = row < a.M ? row : a.M - 1;
            const int wr = first_n + w_row16<FN>(t % FN, fr), col = first_n + C * fg + 4 * (t % FN);
            const unsigned char* x = static_cast<const unsigned char*>(a.x) + m * a.ldx;
            const unsigned char* w = static_cast<const unsigned char*>(a.w) + (wr < a.N ? wr : a.N - 1) * a.ldw;
            float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int g = 0; g < WK; g++) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int b = g; b < args.blocks; b += WK) {
                    const int k = b * kBlock + 16 * fg;
                    Operand<EXACT> ow, ox;
                    ow.set(load_codes<false>(w, k, k + 64, a.K));
                    ox.set(load_codes<false>(x, k, k + 64, a.K));
                    const Factor f(args.xs[m * args.ldxs + b], ws[b]);
                    const f32x4 p = product(ow, ox);
#pragma unroll
                    for (int e = 0; e < 4; e++) part[e] = fmaf(p[e] * f.up, f.rest, part[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) sums[e] = g == 0 ? part[e] : sums[e] + part[e];
            }
            if (row < a.M && col < a.N) finish<TO>(a, row, col, sums);
        }
    };
    auto finish_tile = [&]() __attribute__((always_inline)) {
        if (lost()) {
            once_more();
            stores = 0;  // (of a number that nothing counts)
            return;
        }
        const bool plain = !a.bias && a.act == IRODORI_ACT_NONE && !a.gate && !a.residual;
        if constexpr (!AHEAD) {
            stores = tile.rows_m == BM && tile.rows_n == BN ? 2 * FM : 0;
            if (!stores) {
#pragma unroll
                for (int j = 0; j < FM; j++) {
                    float v[C];
#pragma unroll
                    for (int e = 0; e < C; e++) v[e] = acc[j][e / 4][e % 4];
                    finish_block<TO, false>(a, tile.m0 + wm * TM + 16 * j + fr, tile.n0 + wn * TN + C * fg, lane, v);
                }
            // Behind an epilogue past the L2s: 6000 x 1024 x 2816 with gate and residual 30.4 against 34.3 us, 3000 x 2816 x 1024 22.9 against 23.9,
            // 24000 x 1024 x 2816 96.2 against 97.1.
            } else if (!plain) {
                finish_inner(std::false_type{}, std::true_type{});
            // A Y that the L2s (32 MB) do not hold goes past them: 24000 x 5632 x 1024 154 against 163 us, x 512 92 against 103.
            } else if ((int64_t)a.M * a.N * (int64_t)sizeof(TO) > (32 << 20)) {
                finish_inner(std::true_type{}, std::true_type{});
            } else {
                finish_inner(std::true_type{}, std::false_type{});
            }
        } else if (tile.rows_n == BN) {
            if (!plain) epilogue(std::true_type{});
            store_rows(std::true_type{});
        } else {
            if (!plain) epilogue(std::false_type{});
            store_rows(std::false_type{});
        }
    };
    if constexpr (!AHEAD) {
        for (;;) {
            all_slices();
            finish_tile();  // the next tile's first slices are on their way
            now += stride;
            if (now >= last) return;
            tile = locate(now);
#pragma unroll
            for (int t = 0; t < PRODUCTS; t++) acc[t / FN][t % FN] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 2; i++) {
                pending[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                pending_f[i] = 0.f;
            }
        }
    }

    all_slices();
    // The k groups' sums, added in their order.
    if constexpr (WK > 1) {
        __syncthreads();
        float* part = reinterpret_cast<float*>(smem) + lane;
        constexpr int SUMS = FN * FM * 4 * 64;
        if (wk > 0) {
            float* p = part + ((wk - 1) * WM * WN + wmn) * SUMS;
#pragma unroll
            for (int i = 0; i < FN * FM * 4; i++) p[i * 64] = acc[i / (4 * FN)][i / 4 % FN][i % 4];
        }
        __syncthreads();
        if (wk == 0) {
#pragma unroll
            for (int g = 0; g < WK - 1; g++) {
                const float* p = part + (g * WM * WN + wmn) * SUMS;
#pragma unroll
                for (int i = 0; i < FN * FM * 4; i++) acc[i / (4 * FN)][i / 4 % FN][i % 4] += p[i * 64];
            }
        }
    }
    if (WK > 1 && wk > 0) return;

    finish_tile();
}

// ---- few rows ---------------------------------------------------------------------------------
// M <= 16 rows: a workgroup takes 16 columns of Y, its wavefronts share K's blocks and are summed through LDS.  W moves HBM ->
// registers, each byte once, 32 codes a lane (lane l: W row l % 16, codes 32 (l / 16) .. + 31 of a block), and is multiplied in four 16x16
// steps of 8 of them; X, the B operand, comes from L2.  Bound by reading W.  (The scales are multiplied after the products' loads, not between them:
// 16 x 30000 x 4096 34.8 us against 43.9.)
constexpr int kRowWaves = 8;
template <typename TO>
__global__ __launch_bounds__(64 * kRowWaves) void linear_fp8_rows_kernel(LinearFp8Args args) {
    const LinearArgs& a = args.l;
    constexpr int NW = kRowWaves, U = 4;  // blocks in flight
    __shared__ float sums[NW][16][20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, r = lane & 15, piece = lane >> 4;
    const int n = n0 + r < a.N ? n0 + r : a.N - 1, m = r < a.M ? r : a.M - 1;  // (past them sums that are never stored)
    const unsigned char* w = static_cast<const unsigned char*>(a.w) + (int64_t)n * a.ldw;
    const unsigned char* x = static_cast<const unsigned char*>(a.x) + (int64_t)m * a.ldx;
    const float* xs = args.xs + (int64_t)m * args.ldxs;
    const uniform_ptr ws = uniform(args.ws + (int64_t)(n0 / kBlock) * args.ldws);
    const int b0 = (int)((int64_t)args.blocks * wave / NW), b1 = (int)((int64_t)args.blocks * (wave + 1) / NW);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto run = [&](int b, auto whole, auto count) {
        constexpr int N = decltype(count)::value;
        i32x8 vw[N], vx[N];
        float sx[N], sw[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int k = (b + i) * kBlock + 32 * piece;
            vw[i] = load_codes<decltype(whole)::value>(w, k, k + 16, a.K);
            vx[i] = load_codes<decltype(whole)::value>(x, k, k + 16, a.K);
            sx[i] = xs[b + i];
            sw[i] = ws[b + i];
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            Operand<true> ow, ox;
            ow.set(vw[i]);
            ox.set(vx[i]);
            f32x4 p = product(ow, ox);
            float f = sx[i] * sw[i];
            if (__builtin_expect(any_lane(!normal(f)), false)) {
                const Factor s(sx[i], sw[i]);
                p *= s.up;
                f = s.rest;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] = fmaf(p[e], f, acc[e]);
        }
    };
    const int whole = a.K / kBlock < b1 ? a.K / kBlock : b1;  // blocks with all of their codes
    int b = b0;
    for (; b + U <= whole; b += U) run(b, std::true_type{}, std::integral_constant<int, U>{});
    for (; b < whole; b++) run(b, std::true_type{}, std::integral_constant<int, 1>{});
    for (; b < b1; b++) run(b, std::false_type{}, std::integral_constant<int, 1>{});

    // acc[e]: row m = r, column 4 piece + e.
    *reinterpret_cast<float4*>(&sums[wave][r][4 * piece]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    const int mm = threadIdx.x >> 2, c = 4 * (threadIdx.x & 3);
    if (threadIdx.x >= 64 || mm >= a.M || n0 + c >= a.N) return;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NW; q++) {
        const float4 p = *reinterpret_cast<const float4*>(&sums[q][mm][c]);
        v[0] += p.x;
        v[1] += p.y;
        v[2] += p.z;
        v[3] += p.w;
    }
    finish<TO>(a, mm, n0 + c, v);
}

template <typename TO>
int launch_rows(const LinearFp8Args& a, hipStream_t st, bool go) {
    const int64_t wgs = ((int64_t)a.l.N + 15) / 16;
    if (wgs * (64 * kRowWaves) > UINT32_MAX) return -1;
    if (go) linear_fp8_rows_kernel<TO><<<(unsigned)wgs, 64 * kRowWaves, 0, st>>>(a);
    return 0;
}

constexpr int kResident = 256;  // workgroups of the large tiles: one a CU
template <typename TO, int BM, int BN, int WM, int WN, int WK, int STAGES, bool ASYNC, bool AHEAD, int EU>
int launch_tiles(const LinearFp8Args& a, hipStream_t st, bool go) {
    constexpr int THREADS = 64 * WM * WN * WK;
    const int64_t tiles = (int64_t)((a.l.M + BM - 1) / BM) * ((a.l.N + BN - 1) / BN);
    if (tiles * THREADS > UINT32_MAX) return -1;
    const int64_t wgs = AHEAD || tiles < kResident ? tiles : kResident;
    if (go) linear_fp8_kernel<TO, BM, BN, WM, WN, WK, STAGES, ASYNC, AHEAD, EU><<<(unsigned)wgs, THREADS, 0, st>>>(a);
    return 0;
}

// The tiles a launch takes: of these, the one whose busiest CU is done first, by the microseconds of a tile (f + a a block of K) fitted to
// all tiles' times at 110 sizes (16-bit outputs) and 90 (f32): M from 17 to 30 000, N from 64 to 7360, K from 128 to 3680.  On 50 (40)
// others the choice loses 1.2 % (0.6 %) on the best of them on average, 17 % (13 %) at most.  Tiles that share a CU overlap where they
// wait (rounds count in parts).  E.g. in bf16 with 64 x 64 / 96 x 64 / 128 x 128 / 128 x 256 / 192 x 256 / 256 x 256 tiles: 1500 x 1024 x 2816
// 12.3 / 10.8 / 16.2 / 24.4 / 31.5 / 39 us, 12000 x 1280 x 2816 84 / - / 79 / 53 / 63 / 50, 24000 x 5632 x 1024 327 / - / 253 / 170 / 151 / 156,
// 8192^3 934 / - / 987 / 612 / 533 / 483; into f32 with 64 x 64 / 96 x 64 / 64 x 128 / 128 x 128 1500 x 1024 x 2816 17.0 / 14.9 / 16.2 / 25.9.
struct TileCost {
    int bm, bn;
    float f, a;
    int parts;
    float alone;
};
constexpr TileCost kTiles16[] = {{32, 32, 0.761f, 0.0915f, 4, 1.f},  {64, 64, 0.81f, 0.182f, 1, 1.08f},   {96, 64, 1.833f, 0.2393f, 1, 1.f},
                                 {128, 128, 1.04f, 0.4946f, 1, 1.f}, {128, 256, 0.832f, 0.9837f, 1, 0.93f}, {192, 256, 1.41f, 1.2633f, 1, 1.f},
                                 {256, 256, 2.939f, 1.7536f, 1, 1.f}};
constexpr TileCost kTiles32[] = {{32, 32, 1.254f, 0.0789f, 4, 1.36f}, {64, 64, 1.197f, 0.2262f, 1, 1.f}, {96, 64, 1.466f, 0.4601f, 1, 1.f},
                                 {64, 128, 1.883f, 0.4832f, 1, 1.f},  {128, 128, 1.171f, 0.9313f, 1, 1.f}};
template <int N>
int best_tiles(const TileCost (&t)[N], const LinearFp8Args& a) {
    constexpr int CUS = 256;
    int best = 0;
    double least = 0.;
    for (int i = 0; i < N; i++) {
        const int64_t n = ((int64_t)(a.l.M + t[i].bm - 1) / t[i].bm) * ((a.l.N + t[i].bn - 1) / t[i].bn);
        const double rounds = n <= CUS ? t[i].alone : (double)((n * t[i].parts + CUS - 1) / CUS) / t[i].parts;
        const double c = rounds * (t[i].f + (double)t[i].a * a.blocks);
        if (i == 0 || c < least) {
            least = c;
            best = i;
        }
    }
    return best;
}

}  // namespace

template <typename TO>
int launch_linear_fp8(const LinearFp8Args& a, hipStream_t st, bool go) {
    const LinearArgs& l = a.l;
    if (l.M <= 16) return launch_rows<TO>(a, st, go);
    // The buffer-to-LDS loads take dword-aligned rows, and windows of a tile's rows below 2^31 bytes.
    constexpr int64_t FAR = (int64_t)1 << 22;
    const bool async = !((reinterpret_cast<uintptr_t>(l.x) | reinterpret_cast<uintptr_t>(l.w) | l.ldx | l.ldw) & 3) && l.ldx <= FAR &&
                       l.ldw <= FAR && l.K <= FAR && a.ldxs * 4 <= FAR && a.ldws * 4 <= FAR && l.ldy <= FAR && l.ldr <= FAR;
    if (!async) {
        // Through registers: 64 x 64 against 128 x 128 tiles 11.3 / 15.4 us at 500 x 1024 x 1001 (128 tiles of 64), 33.7 / 16.1 at 1536 x 2048
        // (768), 1115 / 422 at 20000 x 5632 (159 where K is 1000): the smaller ones while they all run at once.
        if (((int64_t)l.M + 63) / 64 * ((l.N + 63) / 64) <= 256) return launch_tiles<TO, 64, 64, 2, 2, 2, 2, false, true, 2>(a, st, go);
        return launch_tiles<TO, 128, 128, 4, 2, 1, 2, false, true, 2>(a, st, go);
    }
    if constexpr (sizeof(TO) == 4) {
        switch (best_tiles(kTiles32, a)) {
            case 0: return launch_tiles<TO, 32, 32, 1, 1, 4, 2, true, true, 2>(a, st, go);
            case 1: return launch_tiles<TO, 64, 64, 1, 2, 2, 2, true, true, 2>(a, st, go);
            case 2: return launch_tiles<TO, 96, 64, 2, 2, 2, 2, true, true, 2>(a, st, go);
            case 3: return launch_tiles<TO, 64, 128, 2, 2, 2, 2, true, true, 2>(a, st, go);
            default: return launch_tiles<TO, 128, 128, 4, 2, 1, 2, true, true, 2>(a, st, go);
        }
    } else {
        switch (best_tiles(kTiles16, a)) {
            case 0: return launch_tiles<TO, 32, 32, 1, 1, 4, 2, true, true, 2>(a, st, go);
            case 1: return launch_tiles<TO, 64, 64, 2, 2, 2, 2, true, true, 4>(a, st, go);
            case 2: return launch_tiles<TO, 96, 64, 2, 2, 2, 3, true, true, 2>(a, st, go);
            case 3: return launch_tiles<TO, 128, 128, 4, 2, 1, 3, true, true, 2>(a, st, go);
            case 4: return launch_tiles<TO, 128, 256, 2, 4, 1, 2, true, false, 2>(a, st, go);
            case 5: return launch_tiles<TO, 192, 256, 2, 4, 1, 2, true, false, 2>(a, st, go);
            default: return launch_tiles<TO, 256, 256, 2, 4, 1, 2, true, false, 2>(a, st, go);
        }
    }
}

template int launch_linear_fp8<bf16>(const LinearFp8Args&, hipStream_t, bool);
template int launch_linear_fp8<f16>(const LinearFp8Args&, hipStream_t, bool);
template int launch_linear_fp8<float>(const LinearFp8Args&, hipStream_t, bool);

}  // namespace irodori
