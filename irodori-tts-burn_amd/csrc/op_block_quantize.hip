// Quantization to e4m3 with a scale for each block of 128 (irodori_op_block_quantize): a row's blocks (the operands of
// irodori_op_linear_fp8's x, behind a gated activation where there is one), or blocks of 128 x 128 (its w).
//
// HBM-bound.  16 lanes take a block of 128 columns, 8 neighbouring elements each: the block's largest magnitude is a maximum
// over a row of lanes, and the codes leave as 128 neighbouring bytes; four blocks' loads are on their way at once.
//
// Measured a call, host side included (floor at a large copy's 5.1 TB/s in brackets): silu(a) b of 8 x 2816 bf16 7.3 us (the call; 4.9 of
// kernel), of 24000 x 2816 64 [67: a copy writes half of its bytes, this a fifth], a 5632 x 1024 f32 weight 8.4 [5.6] (352 workgroups: latency).
#include "common.hpp"
#include "fp8_block.hpp"
#include "linear_tile.hpp"
#include "op_util.hpp"

using namespace irodori;

namespace {

struct QuantArgs {
    const void* x;
    uint8_t* q;
    float* s;
    int64_t ldx, ldq, lds;
    int rows, dim, blocks, act;
    unsigned total, div_blocks;  // rows * blocks; floor(2^32 / blocks)
};

constexpr int kAhead = 4;  // blocks that 16 lanes have in flight

// Blocks are numbered along the rows; a workgroup takes 16 kAhead in a row.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
    const int group = threadIdx.x >> 4, l = threadIdx.x & 15;
    Raw8<T> xa[kAhead], xb[GATED ? kAhead : 1];
    int row[kAhead], at[kAhead], n[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
        const unsigned id = blockIdx.x * (16u * kAhead) + u * 16 + group;
        // The quotient by way of the reciprocal rounded down is at most one short.
        unsigned r = __umulhi(id, a.div_blocks);
        unsigned b = id - r * a.blocks;
        if (b >= (unsigned)a.blocks) {
            b -= a.blocks;
            r++;
        }
        row[u] = r;
        at[u] = b * kBlock + 8 * l;
        n[u] = id < a.total ? a.dim - at[u] : 0;
        const T* x = static_cast<const T*>(a.x) + (int64_t)row[u] * a.ldx + at[u];
        xa[u] = load_raw8(x, n[u]);
        if constexpr (GATED) xb[u] = load_raw8(x + a.dim, n[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
        float v[8];
        to_f32x8(xa[u], v);
        activate<float>(v, a.act);
        if constexpr (GATED) {
            float g[8];
            to_f32x8(xb[u], g);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] *= g[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n[u] ? v[i] : 0.f;
        float amax = row16_max(abs_max(v));
        if (!(amax < __builtin_inff())) amax = row16_max(finite_abs_max(v));
        const float s = scale_of(amax);
        if (n[u] <= 0) continue;
        store_codes8(a.q + row[u] * a.ldq + at[u], n[u], codes8(v, s));
        if (l == 0) a.s[row[u] * a.lds + at[u] / kBlock] = s;
    }
}

// A block of 128 x 128 a workgroup, 8 rows a lane.
template <typename T>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(QuantArgs a) {
    __shared__ float most[2][4];
    const int group = threadIdx.x >> 4, l = threadIdx.x & 15, wave = threadIdx.x >> 6;
    const int tile = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks;
    const int at = block * kBlock + 8 * l, n = a.dim - at;
    Raw8<T> x[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const int row = tile * kBlock + u * 16 + group;
        x[u] = load_raw8(static_cast<const T*>(a.x) + (int64_t)row * a.ldx + at, row < a.rows ? n : 0);
    }
    auto over_block = [&](int slot, auto each) {
        float m = 0.f;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            float v[8];
            to_f32x8(x[u], v);
            m = fmaxf(m, each(v));
        }
        m = wave_max(m);
        if ((threadIdx.x & 63) == 0) most[slot][wave] = m;
        __syncthreads();
        return fmaxf(fmaxf(most[slot][0], most[slot][1]), fmaxf(most[slot][2], most[slot][3]));
    };
    float amax = over_block(0, [](const float (&v)[8]) { return abs_max(v); });
    if (!(amax < __builtin_inff())) amax = over_block(1, [](const float (&v)[8]) { return finite_abs_max(v); });
    const float s = scale_of(amax);
    if (threadIdx.x == 0) a.s[tile * a.lds + block] = s;
    if (n <= 0) return;
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const int row = tile * kBlock + u * 16 + group;
        if (row >= a.rows) continue;
        float v[8];
        to_f32x8(x[u], v);
        store_codes8(a.q + row * a.ldq + at, n, codes8(v, s));
    }
}

int check_quantize(const irodori_block_quantize_desc* dp) {
    IRO_REQUIRE(dp, IRODORI_ERR_INVALID_ARG, "irodori_op_block_quantize: null description");
    const irodori_block_quantize_desc& d = *dp;
    IRO_REQUIRE(op_dtype_ok(d.dtype), IRODORI_ERR_DTYPE, "irodori_op_block_quantize: dtype must be F32, BF16 or F16");
    IRO_REQUIRE(d.rows > 0 && d.dim > 0, IRODORI_ERR_SHAPE, "irodori_op_block_quantize: dims must be positive");
    IRO_REQUIRE(d.rows <= 1 << 28 && d.dim <= 1 << 28, IRODORI_ERR_SHAPE, "irodori_op_block_quantize: dims must be at most 2^28");
    IRO_REQUIRE(d.block_rows == 1 || d.block_rows == kBlock, IRODORI_ERR_CONFIG, "irodori_op_block_quantize: block_rows must be 1 or 128");
    IRO_REQUIRE(d.activation >= IRODORI_ACT_NONE && d.activation <= IRODORI_ACT_GELU_TANH, IRODORI_ERR_CONFIG,
                "irodori_op_block_quantize: unknown activation");
    IRO_REQUIRE(d.block_rows == 1 || (d.activation == IRODORI_ACT_NONE && !d.gated), IRODORI_ERR_CONFIG,
                "irodori_op_block_quantize: blocks of 128 rows take no activation and no gate");
    IRO_REQUIRE(d.ldx >= 0 && d.ldq >= d.dim && d.lds >= blocks_of(d.dim), IRODORI_ERR_SHAPE,
                "irodori_op_block_quantize: ldq must be at least dim, lds at least its blocks of 128, ldx not negative");
    const int64_t most = (int64_t)1 << 32;
    IRO_REQUIRE(d.ldx <= most && d.ldq <= most && d.lds <= most, IRODORI_ERR_SHAPE, "irodori_op_block_quantize: a row stride above 2^32");
    return IRODORI_OK;
}

// q or the scales over x or over one another.
bool outputs_overlap(const irodori_block_quantize_desc& d, const QuantArgs& a) {
    const int64_t nr[3] = {d.rows, 1, 1}, ns[3] = {((int64_t)d.rows + d.block_rows - 1) / d.block_rows, 1, 1};
    const int64_t sx[3] = {d.ldx}, sq[3] = {d.ldq}, ss[3] = {d.lds};
    const Box x(a.x, dtype_bytes(d.dtype), nr, sx, (int64_t)d.dim * (d.gated ? 2 : 1)), q(a.q, 1, nr, sq, d.dim),
        s(a.s, 4, ns, ss, a.blocks);
    return overlap(q, x) || overlap(s, x) || overlap(q, s);
}

template <typename T>
int launch(const irodori_block_quantize_desc& d, QuantArgs& a, hipStream_t st, bool go) {
    if (d.block_rows == kBlock) {
        const int64_t wgs = ((int64_t)d.rows + kBlock - 1) / kBlock * a.blocks;
        if (wgs > UINT32_MAX / 256) return -1;
        if (go) quantize_tiles_kernel<T><<<(unsigned)wgs, 256, 0, st>>>(a);
        return 0;
    }
    const int64_t total = (int64_t)d.rows * a.blocks, wgs = (total + 16 * kAhead - 1) / (16 * kAhead);
    if (wgs > UINT32_MAX / 256) return -1;
    a.total = (unsigned)total;
    a.div_blocks = a.blocks == 1 ? UINT32_MAX : (unsigned)((1ull << 32) / a.blocks);
    if (!go) return 0;
    if (d.gated) quantize_rows_kernel<T, true><<<(unsigned)wgs, 256, 0, st>>>(a);
    else quantize_rows_kernel<T, false><<<(unsigned)wgs, 256, 0, st>>>(a);
    return 0;
}

}  // namespace

extern "C" {

int irodori_op_block_quantize(const irodori_block_quantize_desc* desc, const void* x, uint8_t* q, float* scales, void* stream) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_quantize(desc));
    const irodori_block_quantize_desc& d = *desc;
    IRO_REQUIRE(x && q && scales, IRODORI_ERR_INVALID_ARG, "irodori_op_block_quantize: null argument");
    IRO_REQUIRE(aligned_to(x, dtype_bytes(d.dtype)) && aligned_to(scales, 4), IRODORI_ERR_INVALID_ARG,
                "irodori_op_block_quantize: an argument is not aligned to its element type");
    hipStream_t st = static_cast<hipStream_t>(stream);
    IRO_TRY(check_op_stream(st, "irodori_op_block_quantize"));
    QuantArgs a{x, q, scales, d.ldx, d.ldq, d.lds, d.rows, d.dim, blocks_of(d.dim), d.activation, 0u, 0u};
    const bool apart = !outputs_overlap(d, a);
    int rc;
    if (d.dtype == IRODORI_DTYPE_F32) rc = launch<float>(d, a, st, apart);
    else if (d.dtype == IRODORI_DTYPE_BF16) rc = launch<bf16>(d, a, st, apart);
    else rc = launch<f16>(d, a, st, apart);
    IRO_REQUIRE(rc == 0, IRODORI_ERR_SHAPE, "irodori_op_block_quantize: too many blocks for one launch");
    IRO_REQUIRE(apart, IRODORI_ERR_INVALID_ARG, "irodori_op_block_quantize: an output overlaps another argument");
    return check_launch("block quantize");
    IRO_GUARD_END
}

}  // extern "C"
