// The norms around a block (irodori_op_block_norm): the block's output normed, gated and added to the
// residual stream, and the next block's normed input from the sum, in one pass over the row.
//
//   r = a x + g (N_b(branch) w_b + b_b),  x_out = r,  h = (N(r) w + b) (1 + scale) + shift,  g = branch_scale * gate
//   N(v) = v / sqrt(mean(v^2) + eps)  or  (v - mean(v)) / sqrt(var(v) + eps)
//
// HBM-bound: a row is read once into registers (8 neighbouring elements a lane and chunk), its sums are formed
// there, and it is written once; h is formed from the unrounded r.  Rows of up to 2048 take a wavefront (a reduction is then a
// dozen VALU operations and no barrier), wider ones as many wavefronts as it takes.  The weights and the modulation come from L2 under
// the reductions.
//
// Measured a call, host side included (floor at a large copy's 5.1 TB/s in brackets): 4 x 1280 bf16 7.5 us (the call; 5.2 of kernel),
// 253 x 1280 f32 7.5 (the call; 4.9 of kernel), 1500 x 1024 with gate and modulation into codes 8.2 [3.3] (8.1 of kernel: 375 workgroups, two
// chains of load, reduction and load, of which the second's loads could go out with the first's), 24000 x 1280 around an f32 stream 75 [72].
// Other widths, 24000 rows of bf16 around an f32 stream with gate and modulation: 64 16.8 [3.6] and 333 37.7 [18.8] (most lanes idle),
// 1024 68 [58], 2048 135 [116], 2816 190 [159], 3680 240 [208], 5632 440 [318] (4 chunks a lane: two wavefronts a SIMD, and with several wavefronts a row
// 36 bytes of scratch a lane); 6000 x 16384 327 [231].
#include "common.hpp"
#include "fp8_block.hpp"
#include "op_util.hpp"

using namespace irodori;

namespace {

constexpr int kMostDim = 16384;  // 8 wavefronts of 4 chunks

struct NormArgs {
    const void *x, *branch;
    const float *branch_weight, *branch_bias, *gate, *weight, *bias, *scale, *shift;
    void *x_out, *h;
    float* h_scales;
    int64_t ldx, ldb, ldxo, ldh, ldhs, ldm;
    int rows, dim, mod_rows, branch_norm, norm;
    float branch_eps, eps, stream_scale, branch_scale;
};

// Sum over the wavefront, on the VALU.
__device__ __forceinline__ float sum64(float v) {
    v = row16_sum(v);
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, (unsigned)a[0]) + __builtin_bit_cast(float, (unsigned)a[1]);
    const unsigned w = __builtin_bit_cast(unsigned, v);
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __builtin_bit_cast(float, (unsigned)b[0]) + __builtin_bit_cast(float, (unsigned)b[1]);
}

// A row's sums over its wavefronts: through LDS where it has several, each call with a slot of its own.
template <bool ONE>
struct RowSum {
    float2 (*slots)[8];
    int waves, used = 0;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        a = sum64(a);
        b = sum64(b);
        if constexpr (!ONE) {
            if ((threadIdx.x & 63) == 0) slots[used][threadIdx.x >> 6] = make_float2(a, b);
            __syncthreads();
            a = b = 0.f;
            for (int i = 0; i < waves; i++) {
                a += slots[used][i].x;
                b += slots[used][i].y;
            }
            used++;
        }
        return make_float2(a, b);
    }
};
constexpr int kSlots = 12;  // two norms, three sums each, each formed twice at most

// The norm of a row as v -> ((v pre - mean) - rest) r.  The mean is that of f32 sums and the rest what they missed: the mean
// of the differences, which are exact where they are small.  Where that rest is more than 1/64 of the differences, as in rows whose
// spread is in their last bits, the variance E d^2 - rest^2 would be a difference of near numbers and the rest's own rounding as large as what it
// leaves: the rest joins the mean, rounded, and the differences are formed again.  They are whole numbers of half steps of f32, their mean
// at most half a step, so rest^2 <= variance; and all 0 where the row is a constant.  Where the sums pass f32's range they are
// formed again from values times 2^-80, of which no sum passes it.
struct Norm {
    float pre = 1.f, mean = 0.f, rest = 0.f, r = 1.f;
    __device__ __forceinline__ float operator()(float v) const {
#pragma clang fp contract(off)
        return (fmaf(v, pre, -mean) - rest) * r;
    }
};
// v is zero from dim on; n: the elements of each chunk.
template <int CH, bool ONE>
__device__ __forceinline__ Norm norm_of(const float (&v)[CH][8], const int (&n)[CH], int kind, int dim, float eps, RowSum<ONE>& sum) {
#pragma clang fp contract(off)  // the mean is the rounded one wherever it stands: what it misses is in `rest`
    Norm f;
    if (kind == IRODORI_NORM_NONE) return f;
    const float inv = 1.f / (float)dim;
    for (int turn = 0; turn < 2; turn++) {
        float square;
        if (kind == IRODORI_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) s = fmaf(v[c][i], f.pre, s);
            f.mean = sum(s, 0.f).x * inv;
            auto differences = [&]() __attribute__((always_inline)) {
                float d1 = 0.f, d2 = 0.f;
#pragma unroll
                for (int c = 0; c < CH; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        float d = fmaf(v[c][i], f.pre, -f.mean);
                        d = i < n[c] ? d : 0.f;
                        d1 += d;
                        d2 = fmaf(d, d, d2);
                    }
                const float2 t = sum(d1, d2);
                f.rest = t.x * inv;
                return t.y;
            };
            float squares = differences();
            if (__builtin_expect(f.rest != 0.f && squares < __builtin_inff() && f.rest * f.rest >= 0x1p-12f * (squares * inv), false)) {
                f.mean += f.rest;
                squares = differences();
            }
            square = squares < __builtin_inff() ? fmaxf(squares * inv - f.rest * f.rest, 0.f) : squares;
        } else {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float d = v[c][i] * f.pre;
                    s = fmaf(d, d, s);
                }
            square = sum(s, 0.f).x * inv;
        }
        const float under = square + eps * f.pre * f.pre;  // (2^-160 is no f32 number, a large eps times it is)
        f.r = under == 0.f ? 0.f : 1.f / sqrtf(under);  // (a small one is 0, and all of a row may be its mean)
        if (square < __builtin_inff() || turn == 1) break;
        f.pre = 0x1p-80f;
    }
    return f;
}

// T: the branch's and h's type, TS: the stream's, CH: chunks of 8 elements a lane.  ONE: a row a wavefront, 4 a workgroup; else a row a
// workgroup.
template <typename T, typename TS, int CH, bool ONE>
__global__ __launch_bounds__(ONE ? 256 : 512) void block_norm_kernel(NormArgs a, int fp8) {
    __shared__ float2 slots[ONE ? 1 : kSlots][8];
    const int t = ONE ? threadIdx.x & 63 : threadIdx.x, width = ONE ? 64 : blockDim.x;
    const int row = ONE ? (int)(blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) : (int)blockIdx.x;
    if (row >= a.rows) return;
    RowSum<ONE> sum{slots, width / 64};

    const TS* x = static_cast<const TS*>(a.x) + row * a.ldx;
    int at[CH], n[CH];
    Raw8<TS> rx[CH];
#pragma unroll
    for (int c = 0; c < CH; c++) {
        at[c] = (c * width + t) * 8;
        n[c] = a.dim - at[c];
        rx[c] = load_raw8(x + at[c], n[c]);
    }
    const int64_t mod = a.mod_rows ? (int64_t)(row / a.mod_rows) * a.ldm : 0;
    // A vector by channel, or the value that stands for one.
    auto vec = [&](const float* p, int c, float none, float (&f)[8]) {
        if (p) {
            const Raw8<float> r = load_raw8(p + at[c], n[c]);
            to_f32x8(r, f);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = none;
        }
    };
    float r[CH][8];
    if (a.branch) {
        const T* y = static_cast<const T*>(a.branch) + row * a.ldb;
        Raw8<T> ry[CH];
#pragma unroll
        for (int c = 0; c < CH; c++) ry[c] = load_raw8(y + at[c], n[c]);
        float wb[CH][8], bb[CH][8], g[CH][8];
#pragma unroll
        for (int c = 0; c < CH; c++) {
            vec(a.branch_weight, c, 1.f, wb[c]);
            vec(a.branch_bias, c, 0.f, bb[c]);
            vec(a.gate ? a.gate + mod : nullptr, c, 1.f, g[c]);
        }
#pragma unroll
        for (int c = 0; c < CH; c++) to_f32x8(ry[c], r[c]);
        const Norm f = norm_of<CH, ONE>(r, n, a.branch_norm, a.dim, a.branch_eps, sum);
#pragma unroll
        for (int c = 0; c < CH; c++) {
            float v[8];
            to_f32x8(rx[c], v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float b = fmaf(f(r[c][i]), wb[c][i], bb[c][i]) * (g[c][i] * a.branch_scale);
                r[c][i] = i < n[c] ? fmaf(v[i], a.stream_scale, b) : 0.f;
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            to_f32x8(rx[c], r[c]);
#pragma unroll
            for (int i = 0; i < 8; i++) r[c][i] *= a.stream_scale;
        }
    }
    if (a.x_out) {
        TS* xo = static_cast<TS*>(a.x_out) + row * a.ldxo;
#pragma unroll
        for (int c = 0; c < CH; c++) store8(xo + at[c], n[c], r[c]);
    }
    if (!a.h) return;
    float w[CH][8], b[CH][8];
#pragma unroll
    for (int c = 0; c < CH; c++) {
        float s[8], d[8];
        vec(a.weight, c, 1.f, w[c]);
        vec(a.bias, c, 0.f, b[c]);
        vec(a.scale ? a.scale + mod : nullptr, c, 0.f, s);
        vec(a.shift ? a.shift + mod : nullptr, c, 0.f, d);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            w[c][i] = fmaf(w[c][i], s[i], w[c][i]);
            b[c][i] = fmaf(b[c][i], s[i], b[c][i]) + d[i];
        }
    }
    const Norm f = norm_of<CH, ONE>(r, n, a.norm, a.dim, a.eps, sum);
#pragma unroll
    for (int c = 0; c < CH; c++) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = fmaf(f(r[c][i]), w[c][i], b[c][i]);
        if (!fp8) {
            store8(static_cast<T*>(a.h) + row * a.ldh + at[c], n[c], v);
            continue;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n[c] ? v[i] : 0.f;
        float amax = row16_max(abs_max(v));  // 16 lanes hold a block
        if (!(amax < __builtin_inff())) amax = row16_max(finite_abs_max(v));
        const float s = scale_of(amax);
        if (n[c] > 0) {
            store_codes8(static_cast<uint8_t*>(a.h) + row * a.ldh + at[c], n[c], codes8(v, s));
            if (t % 16 == 0) a.h_scales[row * a.ldhs + at[c] / kBlock] = s;
        }
    }
}

int check_block_norm(const irodori_block_norm_desc* dp) {
    IRO_REQUIRE(dp, IRODORI_ERR_INVALID_ARG, "irodori_op_block_norm: null description");
    const irodori_block_norm_desc& d = *dp;
    IRO_REQUIRE(op_dtype_ok(d.dtype), IRODORI_ERR_DTYPE, "irodori_op_block_norm: dtype must be F32, BF16 or F16");
    IRO_REQUIRE(d.stream_dtype == d.dtype || d.stream_dtype == IRODORI_DTYPE_F32, IRODORI_ERR_DTYPE,
                "irodori_op_block_norm: stream_dtype must be dtype or F32");
    IRO_REQUIRE(d.h_dtype == d.dtype || d.h_dtype == IRODORI_DTYPE_FP8, IRODORI_ERR_DTYPE,
                "irodori_op_block_norm: h_dtype must be dtype or FP8");
    IRO_REQUIRE(d.rows > 0 && d.dim > 0, IRODORI_ERR_SHAPE, "irodori_op_block_norm: dims must be positive");
    IRO_REQUIRE(d.dim <= kMostDim, IRODORI_ERR_SHAPE, "irodori_op_block_norm: dim must be at most 16384");
    for (int kind : {d.branch_norm, d.norm})
        IRO_REQUIRE(kind >= IRODORI_NORM_NONE && kind <= IRODORI_NORM_LAYER, IRODORI_ERR_CONFIG, "irodori_op_block_norm: unknown norm");
    for (float eps : {d.branch_eps, d.eps})
        IRO_REQUIRE(eps >= 1e-30f && eps <= 1e30f, IRODORI_ERR_CONFIG, "irodori_op_block_norm: eps must be between 1e-30 and 1e30");
    for (float s : {d.stream_scale, d.branch_scale})
        IRO_REQUIRE(std::fabs(s) <= 1e38f, IRODORI_ERR_CONFIG, "irodori_op_block_norm: scales must be at most 1e38 in magnitude");
    IRO_REQUIRE(d.mod_rows >= 0, IRODORI_ERR_SHAPE, "irodori_op_block_norm: mod_rows must not be negative");
    IRO_REQUIRE(d.ldx >= 0 && d.ldb >= 0 && d.ldm >= 0 && d.ldxo >= d.dim && d.ldh >= d.dim && d.ldhs >= blocks_of(d.dim),
                IRODORI_ERR_SHAPE,
                "irodori_op_block_norm: ldxo and ldh must be at least dim, ldhs at least its blocks of 128, ldx, ldb and ldm not negative");
    const int64_t most = (int64_t)1 << 32;
    for (int64_t ld : {d.ldx, d.ldb, d.ldxo, d.ldh, d.ldhs, d.ldm})
        IRO_REQUIRE(ld <= most, IRODORI_ERR_SHAPE, "irodori_op_block_norm: a row stride above 2^32");
    return IRODORI_OK;
}

// An output over something that is read or over another one (x_out may be x).
bool outputs_overlap(const irodori_block_norm_desc& d, const NormArgs& a) {
    const size_t es = dtype_bytes(d.dtype), et = dtype_bytes(d.stream_dtype), eh = d.h_dtype == IRODORI_DTYPE_FP8 ? 1 : es;
    const int64_t nr[3] = {d.rows, 1, 1};
    const int64_t nm[3] = {d.mod_rows ? (d.rows + (int64_t)d.mod_rows - 1) / d.mod_rows : 1, 1, 1};
    auto rows = [&](const void* p, size_t e, int64_t ld, int64_t inner) {
        const int64_t s[3] = {ld};
        return Box(p, e, nr, s, inner);
    };
    auto mods = [&](const float* p) {
        const int64_t s[3] = {d.ldm};
        return Box(p, 4, nm, s, d.dim);
    };
    const int64_t vec = (int64_t)4 * d.dim;
    const Box x = rows(a.x, et, d.ldx, d.dim), out[3] = {rows(a.x_out, et, d.ldxo, d.dim), rows(a.h, eh, d.ldh, d.dim),
                                                        rows(a.h_scales, 4, d.ldhs, blocks_of(d.dim))};
    const Box in[] = {rows(a.branch, es, d.ldb, d.dim), Box(a.branch_weight, vec), Box(a.branch_bias, vec), Box(a.weight, vec),
                      Box(a.bias, vec), mods(a.gate), mods(a.scale), mods(a.shift)};
    for (int i = 0; i < 3; i++) {
        for (const Box& b : in)
            if (overlap(out[i], b)) return true;
        if ((i > 0 || a.x_out != a.x) && overlap(out[i], x)) return true;
        for (int j = 0; j < i; j++)
            if (overlap(out[i], out[j])) return true;
    }
    return false;
}

template <typename T, typename TS>
int launch(const NormArgs& a, int fp8, hipStream_t st, bool go) {
    const int waves = (a.dim + 2047) / 2048, chunks = (a.dim + 512 * waves - 1) / (512 * waves);
    const int64_t threads = waves == 1 ? ((int64_t)a.rows + 3) / 4 * 256 : (int64_t)a.rows * waves * 64;
    if (threads > UINT32_MAX) return -1;
    if (!go) return 0;
    const int per = waves == 1 ? 256 : waves * 64;  // (rows of several wavefronts have 3 or 4 chunks)
    auto run = [&](auto ch) {
        constexpr int CH = decltype(ch)::value;
        if (waves == 1) block_norm_kernel<T, TS, CH, true><<<(unsigned)(threads / per), per, 0, st>>>(a, fp8);
        else if constexpr (CH > 2) block_norm_kernel<T, TS, CH, false><<<(unsigned)(threads / per), per, 0, st>>>(a, fp8);
    };
    switch (chunks) {
        case 1: run(std::integral_constant<int, 1>{}); break;
        case 2: run(std::integral_constant<int, 2>{}); break;
        case 3: run(std::integral_constant<int, 3>{}); break;
        default: run(std::integral_constant<int, 4>{});
    }
    return 0;
}

}  // namespace

extern "C" {

int irodori_op_block_norm(const irodori_block_norm_desc* desc, const void* x, const void* branch, const float* branch_weight,
                          const float* branch_bias, const float* gate, void* x_out, const float* weight, const float* bias,
                          const float* scale, const float* shift, void* h, float* h_scales, void* stream) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_block_norm(desc));
    const irodori_block_norm_desc& d = *desc;
    const bool fp8 = d.h_dtype == IRODORI_DTYPE_FP8;
    IRO_REQUIRE(x && (x_out || h), IRODORI_ERR_INVALID_ARG, "irodori_op_block_norm: null argument (x, or both x_out and h)");
    IRO_REQUIRE(branch || !(branch_weight || branch_bias || gate), IRODORI_ERR_INVALID_ARG,
                "irodori_op_block_norm: a branch's weight, bias or gate without a branch");
    IRO_REQUIRE(h || !(weight || bias || scale || shift), IRODORI_ERR_INVALID_ARG,
                "irodori_op_block_norm: a weight, bias, scale or shift without h");
    IRO_REQUIRE(!h_scales == !(h && fp8), IRODORI_ERR_INVALID_ARG, "irodori_op_block_norm: FP8 codes in h and h_scales go together");
    IRO_REQUIRE(!(gate || scale || shift) == !d.mod_rows, IRODORI_ERR_INVALID_ARG,
                "irodori_op_block_norm: a gate, scale or shift and a positive mod_rows go together");
    const size_t es = dtype_bytes(d.dtype), et = dtype_bytes(d.stream_dtype);
    bool aligned = aligned_to(x, et) && aligned_to(x_out, et) && aligned_to(branch, es) && (fp8 || aligned_to(h, es));
    for (const float* p : {branch_weight, branch_bias, gate, weight, bias, scale, shift, (const float*)h_scales}) aligned = aligned && aligned_to(p, 4);
    IRO_REQUIRE(aligned, IRODORI_ERR_INVALID_ARG, "irodori_op_block_norm: an argument is not aligned to its element type");
    IRO_REQUIRE(x_out != x || d.rows == 1 || d.ldx == d.ldxo, IRODORI_ERR_SHAPE, "irodori_op_block_norm: x in place needs ldx == ldxo");
    hipStream_t st = static_cast<hipStream_t>(stream);
    IRO_TRY(check_op_stream(st, "irodori_op_block_norm"));
    const NormArgs a{x, branch, branch_weight, branch_bias, gate, weight, bias, scale, shift, x_out, h, h_scales,
                     d.ldx, d.ldb, d.ldxo, d.ldh, d.ldhs, d.ldm, d.rows, d.dim, d.mod_rows, d.branch_norm, d.norm,
                     d.branch_eps, d.eps, d.stream_scale, d.branch_scale};
    const bool apart = !outputs_overlap(d, a), f32 = d.stream_dtype == IRODORI_DTYPE_F32;
    int rc;
    if (d.dtype == IRODORI_DTYPE_F32) rc = launch<float, float>(a, fp8, st, apart);
    else if (d.dtype == IRODORI_DTYPE_BF16) rc = f32 ? launch<bf16, float>(a, fp8, st, apart) : launch<bf16, bf16>(a, fp8, st, apart);
    else rc = f32 ? launch<f16, float>(a, fp8, st, apart) : launch<f16, f16>(a, fp8, st, apart);
    IRO_REQUIRE(rc == 0, IRODORI_ERR_SHAPE, "irodori_op_block_norm: too many rows for one launch");
    IRO_REQUIRE(apart, IRODORI_ERR_INVALID_ARG, "irodori_op_block_norm: an output overlaps another argument");
    return check_launch("block norm");
    IRO_GUARD_END
}

}  // extern "C"
