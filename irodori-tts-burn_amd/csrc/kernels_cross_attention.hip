// Cross attention on token-major operands as a caller has them (irodori_op_cross_attention): queries
// of one length, an encoder's keys and values of another, heads sharing a key head in groups, lengths
// and a key mask per batch row.
//
// Per key tile and wavefront (32 rows; a row is one token of one head of the group, so a group's
// heads share every tile that is loaded), on the 32x32 matrix-core shapes:
//   S^T = K Q^T      lane l holds row l % 32 and keys 8a + 4 (l / 32) + c of every 32.
//   softmax          p = exp2(s c - m) in f32, c = scale log2(e).  The reference m is lazy: a row's
//                    first score above -inf sets it, and it moves, with the tile's scores formed again, when a
//                    lane's sum of p over a tile shows a p beyond the slack.
//   O^T += V^T P^T   P^T is the S^T accumulator, rounded to the operand type in the 16-bit forms (the
//                    matrix core's operand; its rounding averages out over the keys as V's own does), and summed as
//                    rounded: 2.3e-3 relative L2 from float64 in bf16 and 2.9e-4 in f16, where the output's rounding
//                    alone is 1.7e-3 and 2.1e-4.  (Two operands to a probability would take half as many products again.)
//                    V^T comes from the row-major tile, 16-bit by the transposing LDS read.
// A tile that the mask empties is not loaded, but for the first step's K where there are two key groups or more, which
// is loaded under the mask's latency on the guess that it counts; in a tile that the mask thins, the masked scores are
// -inf and the masked values, which are not loaded, zero.
//
// Measured a call, host side included (the operator's floor in brackets):
//   8 x 1 token over 8200 ragged keys, 16 heads on 4 of 128 (bf16)   26.1 us [19.5]  memory: the runs stream at 4.5 TB/s for
//                                        21 us, the joining launch takes 5
//   2 x 101 over 37 keys, 16 heads of 64 (f32)    8.1 [0.4]   one chain: mask, tile, 4096 cycles of f32 matrix core, join
//   2 x 750 over 631 masked keys, 16 heads of 64 (bf16)   14.3 [1.7]  384 workgroups, a chain of five steps of about 1.2 us
//                                        (softmax on the VALU, then the products) between 4 us of loads and 2 of joining
//   32 x 750 over 4100 ragged keys, 20 heads of 64 (f16)  460 [219]   VALU 65 % and matrix cores 44 % of the cycles, at the
//                                        1.7 GHz that the card's power leaves; 128-dim heads 855 TFLOP/s (bf16)
#include <type_traits>

#include "attn_util.hpp"
#include "common.hpp"
#include "cross_attention.hpp"

namespace irodori {

namespace {

template <typename T>
constexpr int kTile = sizeof(T) == 2 ? 64 : 32;  // keys
// Lazy-reference slack: 2^16, and 2^15 for f16, whose largest finite value is below 2^16.
template <typename T>
constexpr float kSumMax = std::is_same<T, f16>::value ? 32768.f : 65536.f;

// Beside a larger reference, the rounding that a distance's product is spared could be more than the distance.
constexpr float kVast = 16777216.f;

// 16-byte chunk c of tile row r (ROWB bytes): K is read 32 rows at one chunk, 16-bit V 8 rows at two
// neighbouring chunks, f32 V one row at a time.
template <int ROWB>
__device__ __forceinline__ int kswz(int r, int c) {
    return ROWB == 128 ? c ^ ((r >> 1) & 7) : c ^ (r & 15);
}
template <typename T, int ROWB>
__device__ __forceinline__ int vswz(int r, int c) {
    if (sizeof(T) == 4) return c;
    return ROWB == 128 ? c ^ (2 * ((r >> 1) & 3)) : c ^ (2 * (r & 7));
}

// Waits as builtins, which the compiler's own count of outstanding reads takes into account.
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_all() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// The 8 reduction elements of a lane.
template <typename T>
struct Op8 {
    typedef typename Vec8<T>::type type;
};
template <>
struct Op8<float> {
    typedef f32x8 type;
};
template <typename T>
__device__ __forceinline__ f32x16 mma(typename Op8<T>::type a, typename Op8<T>::type b, f32x16 c) {
    if constexpr (sizeof(T) == 2) {
        return mma32x16(a, b, c);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
// V^T operand, keys 16 g + 8 j + 4 (lane / 32) + 0..3 (j = 0, 1) of dim 32 db + lane % 32.
template <typename T, int DH>
__device__ __forceinline__ typename Op8<T>::type read_v(const unsigned char* tile, int g, int db, int lane) {
    constexpr int ROWB = DH * (int)sizeof(T);
    if constexpr (sizeof(T) == 2) {
        const int i = lane & 15, grp = lane >> 4;
        const int col = 32 * db + 16 * (grp & 1) + 4 * (i & 3);
        auto half = [&](int base) {
            const int row = base + 4 * (grp >> 1) + (i >> 2);
            const unsigned char* p = tile + row * ROWB + (vswz<T, ROWB>(row, col >> 3) << 4) + (col & 7) * 2;
            return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)p);
        };
        struct { i16x4 a, b; } f = {half(16 * g), half(16 * g + 8)};
        return __builtin_bit_cast(typename Op8<T>::type, f);
    } else {
        f32x8 f;
        const float* p = reinterpret_cast<const float*>(tile) + (16 * g + 4 * (lane >> 5)) * DH + 32 * db + (lane & 31);
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = p[(8 * (e >> 2) + (e & 3)) * DH];
        return f;
    }
}

// N operands read from LDS and used, in their order.  In the 16-bit forms two are read ahead of the products; the compiler
// by itself reads one at a time, each with its full latency (483 against 464 us at 32 x 750 x 4100 x 20 heads).
// FENCE: in this order also in f32, where the compiler would hold as many as it can.
template <typename T, int N, bool FENCE = sizeof(T) == 2, typename R, typename U>
__device__ __forceinline__ void read_ahead(R read, U use) {
    constexpr int CH = sizeof(T) == 2 ? 2 : 1;
    static_assert(N % CH == 0, "whole chunks");
    typename Op8<T>::type f[2][CH];
#pragma unroll
    for (int i = 0; i < CH; i++) f[0][i] = read(i);
#pragma unroll
    for (int c = 0; c < N / CH; c++) {
        if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
        if (c + 1 < N / CH)
#pragma unroll
            for (int i = 0; i < CH; i++) f[(c + 1) & 1][i] = read((c + 1) * CH + i);
        if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < CH; i++) use(c * CH + i, f[c & 1][i]);
    }
}

// K operand of reduction step ks: keys 32 kb + fr.
template <typename T, int DH>
__device__ __forceinline__ typename Op8<T>::type read_k(const unsigned char* kt, int kb, int ks, int fr, int fh) {
    constexpr int ROWB = DH * (int)sizeof(T);
    typedef typename Op8<T>::type V8;
    const int r = 32 * kb + fr;
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const V8*>(kt + r * ROWB + (kswz<ROWB>(r, 2 * ks + fh) << 4));
    } else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(kt + r * ROWB + (kswz<ROWB>(r, 4 * ks + 2 * fh) << 4));
        const f32x4 hi = *reinterpret_cast<const f32x4*>(kt + r * ROWB + (kswz<ROWB>(r, 4 * ks + 2 * fh + 1) << 4));
        V8 kf;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            kf[e] = lo[e];
            kf[4 + e] = hi[e];
        }
        return kf;
    }
}

// Validity of KT keys.
template <int KT>
__device__ __forceinline__ unsigned long long mask_bits(const uint8_t* m) {
    typedef unsigned u32x4_b __attribute__((ext_vector_type(4), aligned(1)));
    unsigned long long bits = 0;
#pragma unroll
    for (int i = 0; i < KT / 16; i++) {
        const u32x4_b w = *reinterpret_cast<const u32x4_b*>(m + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned nz = ((((w[j] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[j]) >> 7) & 0x01010101u;
            bits |= (unsigned long long)((nz * 0x01020408u) >> 24 & 0xfu) << (16 * i + 4 * j);
        }
    }
    return bits;
}

// Tiles t0 .. te - 1, at most 64 of them, that hold a valid key, in order: lane i has the i-th one's
// index and its keys' bits.
struct TileWord {
    int t, lo, hi;  // per lane
    int n;          // the same in all
};
template <int KT>
__device__ __forceinline__ TileWord tile_word(const uint8_t* mask, int len, int t0, int te, int lane) {
    const int t = t0 + lane, n = len - t * KT;  // keys from the lane's tile on
    unsigned long long bits = 0ull;
    if (t < te && n >= KT) bits = mask ? mask_bits<KT>(mask + (int64_t)t * KT) : KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1ull;
    const int part = len / KT, rest = len % KT;  // the tile that the keys end in: a byte a lane
    if (rest && part >= t0 && part < te && part < t0 + 64) {
        const unsigned long long b = __ballot(lane < rest && (!mask || mask[(int64_t)part * KT + (lane < rest ? lane : 0)]));
        if (t == part) bits = b;
    }
    const bool on = bits != 0ull;
    const unsigned long long act = __ballot(on);
    const int cnt = __popcll(act), below = __popcll(act & ((1ull << lane) - 1ull));
    const int dest = 4 * (on ? below : cnt + (lane - below));
    TileWord tw;
    tw.t = __builtin_amdgcn_ds_permute(dest, t);
    tw.lo = __builtin_amdgcn_ds_permute(dest, (int)(unsigned)bits);
    tw.hi = __builtin_amdgcn_ds_permute(dest, (int)(unsigned)(bits >> 32));
    tw.n = cnt;
    return tw;
}

// a where on is all ones, b where it is 0: one instruction (the expression itself becomes a compare and a select).
__device__ __forceinline__ float bit_select(int on, float a, float b) {
    return __builtin_bit_cast(float, __builtin_amdgcn_bitop3_b32((unsigned)on, __builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b),
                                                                 0xCA));
}
// a b rounded by itself, not inside a multiply-add.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    const float p = a * b;
    return p;
}
// s + a + b in f32.
__device__ __forceinline__ float add_pair(bf16 a, bf16 b, float s) {
    typedef bf16 P2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(P2{a, b}, P2{1.f, 1.f}, s, false);
}
__device__ __forceinline__ float add_pair(f16 a, f16 b, float s) {
    typedef f16 P2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(P2{a, b}, P2{1.f, 1.f}, s, false);
}

// Keys of batch row b.
__device__ __forceinline__ int row_keys(const CrossArgs& a, int b) {
    int n = a.seq_kv;
    if (a.kv_len) n = a.kv_len[b];
    return n < 0 ? 0 : n < a.seq_kv ? n : a.seq_kv;
}
// Key tiles of the 64 batch rows from b0 on, a lane each.
template <int KT>
__device__ __forceinline__ int lane_tiles(const CrossArgs& a, int b0, int lane) {
    return b0 + lane < a.batch ? (row_keys(a, b0 + lane) + KT - 1) / KT : 0;
}
__device__ __forceinline__ int wave_sum(int v) {  // (beside the float one)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
using irodori::wave_sum;

// A workgroup: QW wavefronts of 32 rows times KW groups that take the tiles in turn and are joined
// through LDS.  Two ring slots of KW K and V tiles, moved HBM -> LDS by buffer_load_dwordx4 ... lds;
// UNAL: through registers, for operands off a dword boundary, with rows too far apart for a window or overlapping.
// Without splits it takes one batch row's keys.  With them, the tiles of all batch rows lie end to end
// and each of a.splits workgroups of a key head and row block takes an equal run of them, of several
// batch rows where they are short; the result for batch row b from workgroup w goes to slot w + b.
template <typename T, int DH, int QW, int KW, int WPE, bool UNAL>
__global__ __launch_bounds__(64 * QW * KW) __attribute__((amdgpu_waves_per_eu(WPE))) void cross_kernel(CrossArgs a,
                                                                                                       int row_blocks) {
    typedef typename Op8<T>::type V8;
    constexpr int NW = QW * KW, KT = kTile<T>, KB = KT / 32, ROWB = DH * (int)sizeof(T), TILE = KT * ROWB;
    constexpr int RPI = 1024 / ROWB, NI = KT / RPI, LPW = KW * NI / NW, DB = DH / 32, CH = ROWB / 16;
    constexpr int RING = 4 * KW * TILE, PER = (DB * 16 + 2) * 64;
    static_assert(LPW * NW == KW * NI && NI % LPW == 0, "a wavefront's loads of a stage lie in one tile");
    static_assert((KW - 1) * QW * PER * 4 <= RING, "the groups' results fit the rings");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[RING];  // K [2][KW][TILE], V [2][KW][TILE]
    constexpr int VOFF = 2 * KW * TILE;

    const int lane = threadIdx.x & 63, fr = lane & 31, fh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int qw = wave % QW, kw = wave / QW;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int rb = id % row_blocks;
    id /= row_blocks;
    const bool split = a.splits > 1;
    int b, hk, w = 0;
    int64_t at = 0, stop = 0;  // split: the run's next tile and its end, in all batch rows' tiles
    if (split) {
        w = id % a.splits;
        hk = id / a.splits;
        int64_t all = 0;
        for (int i = 0; i < a.batch; i += 64) all += wave_sum(lane_tiles<KT>(a, i, lane));
        at = all * w / a.splits;
        stop = all * (w + 1) / a.splits;
        b = 0;
    } else {
        hk = id % a.kv_heads;
        b = id / a.kv_heads;
    }
    // c = 0 would turn a masked key's -inf into NaN: the queries are multiplied by it instead.
    float c = a.scale * 1.4426950408889634f;
    const bool zero = c == 0.f;
    if (zero) c = 1.f;
    const float masked = c > 0.f ? -INFINITY : INFINITY;  // the score that vanishes
    // Load instruction ii of this wave in a stage: rows RPI (row0 + ii) .. of tile `tile` of the step's;
    // lane -> row lane / CH, physical chunk lane % CH.
    const int tile = wave * LPW / NI, part = wave * LPW % NI;
    typedef typename std::conditional<UNAL, int64_t, unsigned>::type Off;  // (a window's stay below 2^31)
    Off voK[LPW], voV[LPW];
#pragma unroll
    for (int ii = 0; ii < LPW; ii++) {
        const int r = (part + ii) * RPI + lane / CH;
        voK[ii] = (Off)(r * (a.ks[1] * (int)sizeof(T))) + (kswz<ROWB>(r, lane % CH) << 4);
        voV[ii] = (Off)(r * (a.vs[1] * (int)sizeof(T))) + (vswz<T, ROWB>(r, lane % CH) << 4);
    }

    int tiles = 0;  // split: those of the lane's batch row among the 64 around b
    for (int64_t before = 0;; b++) {  // batch rows of the run
        int t_begin = 0, t_end;
        if (split) {
            if (at >= stop) return;
            if (b % 64 == 0) tiles = lane_tiles<KT>(a, b, lane);
            t_end = __builtin_amdgcn_readlane(tiles, b & 63);
            const int64_t after = before + t_end;
            if (at >= after) {
                before = after;
                continue;
            }
            t_begin = (int)(at - before);
            if (stop < after) t_end = (int)(stop - before);
            at = before + t_end;
            before = after;
        }
        int rows = a.rows;
        if (a.q_len) {
            const int n = a.q_len[b];
            rows = n <= 0 ? 0 : (n < a.seq_q ? n : a.seq_q) * a.group;
        }
        const int row0 = rb * 32 * QW;
        if (row0 >= rows) {  // rows past the length stay as they were
            if (split) continue;
            return;
        }
        const int len = row_keys(a, b);
        if (!split) t_end = (len + KT - 1) / KT;
        const T* Kb = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
        const T* Vb = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
        const uint8_t* mb = a.mask ? a.mask + b * a.mask_stride : nullptr;
        const int row = row0 + 32 * qw + fr, rc = row < rows ? row : rows - 1;
        const int tok = rc / a.group, head = hk * a.group + (rc - tok * a.group);
        V8 qf[DH / 16];
        {
            typedef T Q8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
            const T* qp = static_cast<const T*>(a.q) + b * a.qs[0] + tok * a.qs[1] + head * a.qs[2] + 8 * fh;
#pragma unroll
            for (int ks = 0; ks < DH / 16; ks++) qf[ks] = __builtin_bit_cast(V8, *reinterpret_cast<const Q8*>(qp + 16 * ks));
            if (zero) {
#pragma unroll
                for (int ks = 0; ks < DH / 16; ks++) qf[ks] *= static_cast<T>(0.f);
            }
        }
        f32x16 o[DB];
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[db][e] = 0.f;
        float m = 0.f, l_run = 0.f;
        bool unset = true;  // m is no reference yet: no tile so far, or only scores of -inf
        bool first = true;  // any lane's unset
        bool vast = false;  // any lane's |m| above kVast

        for (int t0 = t_begin; t0 < t_end; t0 += 64) {
            wait_lds();
            raw_barrier();  // the rings may still be read
            // This wave's share of K tile t, and of V tile t without its masked rows (0 times a masked value's NaN or
            // infinity would not be 0), into ring slot `slot`.  Rows past the last key and those left out read as zero.
            auto load = [&](const T* base, const int64_t token, const Off (&vo)[LPW], int off, int t, int slot, auto kept) {
                const int left = len - t * KT, n = left < KT ? left : KT;  // rows of the tile
                const T* src = base + (int64_t)t * KT * token;
                unsigned char* dst = smem + off + (slot * KW + tile) * TILE + part * 1024;
#pragma unroll
                for (int ii = 0; ii < LPW; ii++) {
                    const int r = (part + ii) * RPI + lane / CH;
                    if constexpr (UNAL) {
                        typedef T E16 __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
                        u32x4 x = {0, 0, 0, 0};
                        if (r < n && kept(r)) x = __builtin_bit_cast(u32x4, *reinterpret_cast<const E16*>(src + vo[ii] / (int)sizeof(T)));
                        *reinterpret_cast<u32x4*>(dst + ii * 1024 + 16 * lane) = x;
                    } else {
                        buf_load_lds16(make_rsrc(src, (unsigned)((n - 1) * token * (int)sizeof(T)) + ROWB), kept(r) ? vo[ii] : 0x80000000u,
                                       dst + ii * 1024);
                    }
                }
            };
            auto load_k = [&](int t, int slot) { load(Kb, a.ks[1], voK, 0, t, slot, [](int) { return true; }); };
            auto load_v = [&](int t, int slot, unsigned lo, unsigned hi) {
                load(Vb, a.vs[1], voV, VOFF, t, slot, [&](int r) { return !mb || (((r < 32 ? lo : hi) >> (r & 31)) & 1u); });
            };
            // Few rows: the first step's K is loaded under the mask's latency, on the guess that its tiles hold a
            // key (many rows want the registers).
            constexpr bool GUESS = KW > 1;
            const int guess = t0 + tile < t_end ? t0 + tile : t_end - 1;
            if (GUESS && mb) load_k(guess, 0);
            const TileWord tw = tile_word<KT>(mb, len, t0, t_end, lane);
            const int nact = tw.n, niter = (nact + KW - 1) / KW;
            if (niter == 0) {  // the same for every wave
                if (GUESS) wait_all();
                continue;
            }
            // Step j's tile that this wave has a share of; entries past the last are clamped to it, so every
            // wave issues the same loads.
            auto load_step = [&](int j, int slot, bool k) {
                int li = j * KW + tile;
                li = li < nact ? li : nact - 1;
                const int t = __builtin_amdgcn_readlane(tw.t, li);
                if (k) load_k(t, slot);
                load_v(t, slot, (unsigned)__builtin_amdgcn_readlane(tw.lo, li), (unsigned)__builtin_amdgcn_readlane(tw.hi, li));
            };
            bool guessed = false;
            if (GUESS && mb) {
                guessed = __builtin_amdgcn_readlane(tw.t, tile < nact ? tile : nact - 1) == guess;
                if (!guessed) wait_all();
            }
            load_step(0, 0, !guessed);
            for (int j = 0; j < niter; j++) {
                // This wave's loads of step j have landed, and its reads of the slot refilled next are done.
                const int slot = j & 1;
                wait_all();
                raw_barrier();
                if (j + 1 < niter) load_step(j + 1, slot ^ 1, true);
                const unsigned char* kt = smem + (slot * KW + kw) * TILE;
                const int li = j * KW + kw;
                if (li >= nact) continue;  // this group has no tile in the last step
                const unsigned char* vt = kt + VOFF;
                const unsigned word[2] = {(unsigned)__builtin_amdgcn_readlane(tw.lo, li),
                                          (unsigned)__builtin_amdgcn_readlane(tw.hi, li)};
                f32x16 s[KB];
                auto scores = [&](auto fence) {
#pragma unroll
                    for (int kb = 0; kb < KB; kb++)
#pragma unroll
                        for (int e = 0; e < 16; e++) s[kb][e] = 0.f;
                    constexpr int KS = DH / 16;
                    read_ahead<T, KB * KS, decltype(fence)::value>([&](int i) { return read_k<T, DH>(kt, i / KS, i % KS, fr, fh); },
                                           [&](int i, V8 f) { s[i / KS] = mma<T>(f, qf[i % KS], s[i / KS]); });
                    if ((KB == 2 ? word[0] & word[1] : word[0]) != 0xffffffffu) {  // keys 32 kb + 8 g + 4 fh + i of this lane
#pragma unroll
                        for (int kb = 0; kb < KB; kb++) {
                            const int wd = (int)(word[kb] >> (4 * fh));
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                s[kb][e] = bit_select(__builtin_amdgcn_sbfe(wd, 8 * (e >> 2) + (e & 3), 1), s[kb][e], masked);
                            }
                        }
                    }
                };
                scores(std::integral_constant<bool, sizeof(T) == 2>{});
                // Largest of the row's scores over the tile, in the softmax's units.
                auto tile_max = [&]() {
                    float mx = -INFINITY;
#pragma unroll
                    for (int kb = 0; kb < KB; kb++)
#pragma unroll
                        for (int e = 0; e < 16; e++) mx = fmaxf(mx, rounded_product(s[kb][e], c));
                    return max_halves(mx);
                };
                if (first) {
                    // (A row whose scores are all -inf so far adds nothing at any m, and must not keep one.)
                    const float t = tile_max();
                    if (unset && t != -INFINITY) {
                        m = t;
                        unset = false;
                    }
                    first = __any(unset);
                    vast = __any(fabsf(m) > kVast);
                }
                // The scores become their distances from the reference, which alone stay live.
                V8 pf[2 * KB];
                auto exps = [&](auto distance) {
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kb = 0; kb < KB; kb++)
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float p = fast_exp2(distance(s[kb][e]));
                            pf[2 * kb + (e >> 3)][e & 7] = static_cast<T>(p);
                            if (sizeof(T) == 4) sum[e & 3] += p;
                        }
                    if constexpr (sizeof(T) == 2) {
                        // As the P V product takes them (so the weights add up to one), two an instruction.
#pragma unroll
                        for (int g = 0; g < 2 * KB; g++)
#pragma unroll
                            for (int i = 0; i < 4; i++) sum[i] = add_pair(pf[g][2 * i], pf[g][2 * i + 1], sum[i]);
                    }
                    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
                };
                float psum = exps([&](float x) { return fmaf(x, c, -m); });
                const unsigned long long over = __ballot(!(psum <= kSumMax<T>));
                if (over || vast) {
                    // Lanes l and l ^ 32 hold one row's two key halves: either one asks for both.
                    const bool need = (((over >> lane) | (over >> (lane ^ 32))) & 1ull) || fabsf(m) > kVast;
                    // The scores are formed again: a distance from a reference far below has lost them in its rounding.  The new
                    // distances are those of rounded products, as the reference is one, so the largest is 0.
                    scores(std::true_type{});
                    const float mx = tile_max(), mn = need ? fmaxf(m, mx) : m, corr = fast_exp2(m - mn);
                    m = mn;
                    vast = __any(fabsf(m) > kVast);
#pragma unroll
                    for (int db = 0; db < DB; db++) o[db] *= corr;
                    l_run *= corr;
                    psum = exps([&](float x) { return rounded_product(x, c) - m; });
                }
                l_run += psum;
                read_ahead<T, 2 * KB * DB>([&](int i) { return read_v<T, DH>(vt, i / DB, i % DB, lane); },
                                           [&](int i, V8 f) { o[i % DB] = mma<T>(f, pf[i / DB], o[i % DB]); });
            }
        }

        // Join the key groups through LDS [group - 1][QW][16 DB + 2][64 lanes] in their order.
        float m_run = unset ? -INFINITY : m;
        if constexpr (KW > 1) {
            float* comb = reinterpret_cast<float*>(smem) + lane;
            __syncthreads();
            if (kw > 0) {
                float* cp = comb + ((kw - 1) * QW + qw) * PER;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int e = 0; e < 16; e++) cp[(16 * db + e) * 64] = o[db][e];
                cp[16 * DB * 64] = m_run;
                cp[(16 * DB + 1) * 64] = l_run;
            }
            __syncthreads();
            if (kw == 0) {
#pragma unroll
                for (int g = 1; g < KW; g++) {
                    const float* cp = comb + ((g - 1) * QW + qw) * PER;
                    const float m1 = cp[16 * DB * 64], l1 = cp[(16 * DB + 1) * 64];
                    const float mt = fmaxf(m_run, m1), mu = mt == -INFINITY ? 0.f : mt;
                    const float c0 = fast_exp2(m_run - mu), c1 = fast_exp2(m1 - mu);
#pragma unroll
                    for (int db = 0; db < DB; db++)
#pragma unroll
                        for (int e = 0; e < 16; e++) o[db][e] = o[db][e] * c0 + cp[(16 * db + e) * 64] * c1;
                    l_run = l_run * c0 + l1 * c1;
                    m_run = mt;
                }
            }
        }

        // o[db][e] = O[row][32 db + 8 (e / 4) + 4 fh + e % 4].
        const float l = sum_halves(l_run);
        if (kw == 0 && row < rows) {
            if (split) {
                const int64_t slot = ((int64_t)hk * (a.splits + a.batch) + w + b) * a.rows + row;
                float* op = a.partial + slot * DH + 4 * fh;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *reinterpret_cast<float4*>(op + 32 * db + 8 * g) =
                            make_float4(o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]);
                float2* ml = reinterpret_cast<float2*>(a.partial + (int64_t)a.kv_heads * (a.splits + a.batch) * a.rows * DH);
                if (fh == 0) ml[slot] = make_float2(m_run, l);
            } else {
                const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
                typedef T O4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
                T* op = static_cast<T*>(a.out) + b * a.os[0] + tok * a.os[1] + head * a.os[2] + 4 * fh;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        O4 v;
#pragma unroll
                        for (int i = 0; i < 4; i++) v[i] = static_cast<T>(o[db][4 * g + i] * inv);
                        *reinterpret_cast<O4*>(op + 32 * db + 8 * g) = v;
                    }
            }
        }
        if (!split) return;
    }
}

// The runs' results of a row joined: a wavefront per row.  Lane i holds the weight exp2(m_i - M) of run i,
// 64 at a time; a lane then sums DH / 64 dimensions.
template <typename T, int DH>
__global__ __launch_bounds__(64) void cross_join_kernel(CrossArgs a) {
    const int lane = threadIdx.x;
    const int row = (int)(blockIdx.x % (unsigned)a.rows), bh = (int)(blockIdx.x / (unsigned)a.rows);
    const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
    const int tok = row / a.group, head = hk * a.group + (row - tok * a.group);
    if (a.q_len && tok >= a.q_len[b]) return;
    int64_t all = 0, before = 0;
    int mine = 0;
    for (int x = 0; x < a.batch; x += 64) {
        const int n = lane_tiles<kTile<T>>(a, x, lane);
        all += wave_sum(n);
        before += wave_sum(x + lane < b ? n : 0);
        if (b - x >= 0 && b - x < 64) mine = __builtin_amdgcn_readlane(n, b - x);
    }
    // Run w holds tiles all w / splits .. all (w + 1) / splits - 1: those from w0 to w1 have some of row b's.
    int w0 = 0, w1 = -1;
    if (mine > 0) {
        w0 = (int)(((before + 1) * a.splits + all - 1) / all) - 1;
        w1 = (int)(((before + mine) * a.splits + all - 1) / all) - 1;
    }
    const int64_t slot0 = ((int64_t)hk * (a.splits + a.batch) + b) * a.rows + row;  // run w's is w rows further
    const float2* ml = reinterpret_cast<const float2*>(a.partial + (int64_t)a.kv_heads * (a.splits + a.batch) * a.rows * DH);
    constexpr int PER = DH / 64;
    float o[PER], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < PER; j++) o[j] = 0.f;
    for (int x = w0; x <= w1; x += 64) {
        const int n = w1 + 1 - x < 64 ? w1 + 1 - x : 64;
        const float* p = a.partial + (slot0 + (int64_t)x * a.rows) * DH + lane;
        constexpr int U = 8;  // runs in flight, the first of them with the weights
        float f[U][PER];
        auto load = [&](int i) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < PER; j++) f[u][j] = i + u < n ? p[(int64_t)(i + u) * a.rows * DH + 64 * j] : 0.f;
        };
        load(0);
        // (Where the batch has fewer tiles than runs, some runs are empty and wrote nothing.)
        const int64_t w = x + lane;
        const bool wrote = lane < n && all * w / a.splits < all * (w + 1) / a.splits;
        const float2 v = wrote ? ml[slot0 + w * a.rows] : make_float2(-INFINITY, 0.f);
        const float mt = fmaxf(m, wave_max(v.x)), mu = mt == -INFINITY ? 0.f : mt;
        const float c0 = fast_exp2(m - mu), weight = wrote ? fast_exp2(v.x - mu) : 0.f;
        const unsigned long long there = __ballot(wrote);
        l = l * c0 + wave_sum(v.y * weight);
        m = mt;
#pragma unroll
        for (int j = 0; j < PER; j++) o[j] *= c0;
        for (int i = 0; i < n; i += U) {
            if (i > 0) load(i);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), (i + u) & 63));
#pragma unroll
                for (int j = 0; j < PER; j++)
                    if (i + u < n && (there >> (i + u) & 1)) o[j] = fmaf(f[u][j], c, o[j]);
            }
        }
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T* op = static_cast<T*>(a.out) + b * a.os[0] + tok * a.os[1] + head * a.os[2];
#pragma unroll
    for (int j = 0; j < PER; j++) op[64 * j + lane] = static_cast<T>(o[j] * inv);
}

template <typename T, int DH, int QW, int KW, int WPE, bool UNAL>
int launch_cfg(const CrossArgs& a, hipStream_t st, bool go) {
    const int rbs = (int)(((int64_t)a.rows + 32 * QW - 1) / (32 * QW));
    const int64_t wgs = (int64_t)rbs * a.kv_heads * (a.splits > 1 ? a.splits : a.batch);
    const int64_t joins = (int64_t)a.batch * a.kv_heads * a.rows;
    if (wgs > UINT32_MAX / (64 * QW * KW) || (a.splits > 1 && joins > UINT32_MAX / 64)) return -1;
    if (!go) return 0;
    cross_kernel<T, DH, QW, KW, WPE, UNAL><<<(unsigned)wgs, 64 * QW * KW, 0, st>>>(a, rbs);
    if (a.splits > 1) cross_join_kernel<T, DH><<<(unsigned)joins, 64, 0, st>>>(a);
    return 0;
}

}  // namespace

// 64-row workgroups of a launch that does not split its keys.
static int64_t row_groups(int batch, int kv_heads, int rows) { return ((int64_t)rows + 63) / 64 * kv_heads * batch; }

// As many workgroups as run at once: at 1 x 16 heads x 1 x 16400 keys (bf16, 64-dim) 4 / 8 / 16 / 32 / 64 runs a head
// take 45 / 28 / 23 / 25 / 31 us, unsplit 141; at 8 x 4 key heads x 1 x 8200 ragged keys (128-dim) 64 / 96 / 128 / 192 take
// 30.6 / 27.3 / 27.2 / 34.3, unsplit 125.  A run has two tiles at least, and the split has to save more than the
// joining kernel's 5 us: about 8 tiles of a workgroup's time.
int cross_splits(bool f32, int batch, int kv_heads, int rows, int seq_kv, int head_dim) {
    const int64_t tiles = (seq_kv + 63) / 64, per_batch = row_groups(1, kv_heads, rows);
    int64_t n = (head_dim == 128 && !f32 ? 512 : 256) / per_batch;
    n = n < batch * tiles / 2 ? n : batch * tiles / 2;
    return n > batch && tiles * (n - batch) > 8 * n ? (int)n : 1;
}

template <typename T, int DH>
int launch_cross(const CrossArgs& a, hipStream_t st, bool go) {
    constexpr int64_t es = sizeof(T);
    constexpr bool F32 = sizeof(T) == 4;
    // Windows of a tile's rows stay below 2^31 bytes, and the buffer-to-LDS loads take dword-aligned rows.  Values
    // whose rows overlap (a stride of 0) have rows past the last key inside the window, where they would not read as zero.
    const bool unal = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 3) ||
                      ((a.ks[0] | a.ks[1] | a.ks[2] | a.vs[0] | a.vs[1] | a.vs[2]) * es & 3) ||
                      a.ks[1] * es > (1 << 24) || a.vs[1] * es > (1 << 24) || a.vs[1] < DH;
    constexpr int SMALL = DH == 64 ? 2 : 1;  // wavefronts per SIMD, of two (one) workgroups a CU
    if (unal) return launch_cfg<T, DH, 2, 2, SMALL, true>(a, st, go);
    // f32 in one block of 32 rows is bound by the matrix cores, most of whose rows are padding: a group on every SIMD
    // (38 against 51 us at 8 x 4 key heads x 1 x 8200; at 128-dim the rings do not fit).
    if constexpr (F32 && DH == 64) {
        if (a.rows <= 32) return launch_cfg<T, DH, 1, 4, 1, false>(a, st, go);
    }
    // Runs of 128-dim heads in two workgroups a CU, which hide each other's ends, rather than one with two
    // key groups (27.2 against 30.0 us at 8 x 4 key heads x 1 x 8200; 64-dim heads fit two a CU either way).
    if constexpr (!F32 && DH == 128) {
        if (a.splits > 1) return launch_cfg<T, DH, 2, 1, 1, false>(a, st, go);
    }
    if (a.splits > 1 || row_groups(a.batch, a.kv_heads, a.rows) <= 256 * SMALL) return launch_cfg<T, DH, 2, 2, SMALL, false>(a, st, go);
    // More workgroups than the one round that fits the chip.  Where a key head has 64 rows at most, wider ones would hold rows
    // that do not exist.  16-bit: two wavefronts, one key group (32 batch rows x 20 heads, one row over 100 / 600 / 4100 keys,
    // 64-dim 7.7 / 19.6 / 130 us, against 8.4 / 22.3 / 134 with 128 rows a workgroup and 10.1 / 23.3 / 156 with two key groups;
    // 10 x 64 x 64 rows over 1000 keys 29, 38, 36 us, 128-dim 76, 82, 84).  f32, bound by the matrix cores: two key groups
    // (128-dim, 32 x 20 x one row over 100 / 600 / 4100 keys 46 / 166 / 979 against 56 / 231 / 1510 us; 64-dim, 128 x 4 x 64 rows
    // over 600 keys 52 against 84).
    if (a.rows <= 64) {
        if constexpr (F32) return launch_cfg<T, DH, 2, 2, SMALL, false>(a, st, go);
        else return launch_cfg<T, DH, 2, 1, SMALL, false>(a, st, go);
    }
    // 128 rows a workgroup with one key group: at 750 queries x 1381 keys x 16 heads (bf16, 64-dim), against 64 rows with two,
    // 21.4 / 27.1 us for 2 batch rows, 34 / 31 for 4, 46 / 55 for 8; 8 heads of 128 dimensions, 4 and 8 batch rows, 31 / 42 and
    // 49 / 64; in f32 186 / 150 and 271 / 291, 128-dim 189 / 203 and 350 / 306; 32 x 20 x 130 rows over 1000 keys 56 / 57, f32
    // 329 / 287.
    return launch_cfg<T, DH, 4, 1, DH == 64 && !F32 ? 3 : 2, false>(a, st, go);
}

template int launch_cross<bf16, 64>(const CrossArgs&, hipStream_t, bool);
template int launch_cross<bf16, 128>(const CrossArgs&, hipStream_t, bool);
template int launch_cross<f16, 64>(const CrossArgs&, hipStream_t, bool);
template int launch_cross<f16, 128>(const CrossArgs&, hipStream_t, bool);
template int launch_cross<float, 64>(const CrossArgs&, hipStream_t, bool);
template int launch_cross<float, 128>(const CrossArgs&, hipStream_t, bool);

}  // namespace irodori
