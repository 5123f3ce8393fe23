// The rotary-position operator (irodori_op_rope): queries and keys of a batch rotated by their
// positions in one launch.
//
// Pair p of a head is (x[2p], x[2p + 1]) (interleaved) or (x[p], x[p + rot / 2]) (halves); with
// angle = position * f_p it becomes A (a cos - b sin, a sin + b cos).  The frequencies are made on
// the host in f64, in turns per position, and ride in the kernel's arguments; a position's turns are
// formed and reduced to half a turn in f64 (at position 2^20 an f32 product is off by 0.06 radians),
// then sine and cosine are f32.
//
// HBM-bound: every element is read and written once.  A workgroup takes some tokens and some of
// their heads; it issues all of its loads, then makes the tokens' cosines and sines (one per pair,
// shared by all heads) in LDS under their latency, then rotates and stores.  Measured a call, host side
// included (floor at a large copy's 4.9 TB/s in brackets): 8 tokens of 20 128-dim heads 7.8 us (the launch;
// 4.4 of kernel), 2 x 750 x 32 heads in f32 7.6 [5.0], 8 x 4001 ragged tokens x 40 heads in bf16 59 [48], 44 us of
// kernel where the inputs are in the last-level cache.  Stores past the caches lost (60.6 against 58.9).
#include "common.hpp"
#include "op_util.hpp"

using namespace irodori;

namespace {

constexpr int kMaxRot = 512;   // rotating dimensions of a head: 256 frequencies, 2 KB of arguments
constexpr int kMaxDim = 1024;  // of a head
constexpr int kItems = 4;      // units a thread holds
constexpr int kTable = 2048;   // cosine / sine pairs of a workgroup (16 KB of LDS)

struct RopeSide {
    const void* x;
    void* y;
    int64_t xs[3], ys[3];  // batch, token, head strides in elements
    int heads, rot_heads;
};
struct RopeArgs {
    RopeSide q, k;
    const int32_t* positions;
    const int32_t* lengths;
    int first_pos, batch, seq, pairs;
    int units;          // units of a head: vectors of pairs, then vectors that pass through
    int rot_units;      // of them with pairs
    int tokens, heads;  // per workgroup
    int tok_blocks, head_blocks;
    unsigned div_units, div_heads;  // ceil(2^32 / d), for d > 1: exact quotients of the workgroup's unit indexes
    float amplitude, sin_sign;
    double turns[kMaxRot / 2];
};

// V elements at an address aligned to the element.
template <typename T, int V>
struct Pack {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <typename T>
struct Pack<T, 1> {
    typedef T type;
};
// A unit is two packs of V: an interleaved unit covers elements 2 V u .. 2 V u + 2 V - 1 (V pairs),
// a halves unit V u .. and the same past rot / 2; a unit that passes through covers 2 V elements too.
template <typename T, int V, bool HALVES>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    typedef typename Pack<T, V>::type P;
    __shared__ float2 table[kTable];
    const int tid = threadIdx.x;
    int id = blockIdx.x;
    const int hb = id % a.head_blocks;
    id /= a.head_blocks;
    const int tb = id % a.tok_blocks, b = id / a.tok_blocks;
    const int s0 = tb * a.tokens, h0 = hb * a.heads;
    int len = a.seq;
    if (a.lengths) {
        const int n = a.lengths[b];  // (below 0 none: len - s0 must not leave 32 bits)
        len = n < 0 ? 0 : n < len ? n : len;
    }
    const int nt = len - s0 < a.tokens ? len - s0 : a.tokens;
    if (nt <= 0) return;  // rows past the length stay as they were
    const int ht = a.q.heads + a.k.heads;
    const int nh = ht - h0 < a.heads ? ht - h0 : a.heads;
    const int half = a.pairs;  // rot / 2

    P lo[kItems], hi[kItems];
    int where[kItems];  // token << 16 | unit, or -1
    T* dst[kItems];
    bool turn[kItems];
#pragma unroll
    for (int i = 0; i < kItems; i++) {
        const unsigned it = i * 256 + tid;
        const unsigned hu = a.units == 1 ? it : __umulhi(it, a.div_units);  // it / units
        const int u = (int)(it - hu * a.units);
        const unsigned t = a.heads == 1 ? hu : __umulhi(hu, a.div_heads);
        const int h = h0 + (int)(hu - t * a.heads);
        where[i] = -1;
        if ((int)t >= nt || h >= h0 + nh) continue;
        const bool is_k = h >= a.q.heads;
        const RopeSide& s = is_k ? a.k : a.q;
        const int hh = is_k ? h - a.q.heads : h;
        turn[i] = u < a.rot_units && hh < s.rot_heads;
        // In place, what passes through is there already.
        if (!turn[i] && s.x == s.y) continue;
        const int e = HALVES && u < a.rot_units ? V * u : 2 * V * u;
        const int step = HALVES && u < a.rot_units ? half : V;
        const T* src = static_cast<const T*>(s.x) + b * s.xs[0] + (int64_t)(s0 + (int)t) * s.xs[1] + hh * s.xs[2] + e;
        dst[i] = static_cast<T*>(s.y) + b * s.ys[0] + (int64_t)(s0 + (int)t) * s.ys[1] + hh * s.ys[2] + e;
        lo[i] = *reinterpret_cast<const P*>(src);
        hi[i] = *reinterpret_cast<const P*>(src + step);
        where[i] = (int)(t << 16) | u;
    }
    for (int i = tid; i < nt * a.pairs; i += 256) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        const int s = s0 + t;
        const int pos = a.positions ? a.positions[(int64_t)b * a.seq + s] : a.first_pos + s;
        const double r = (double)pos * a.turns[p];
        float sn, cs;
        sincospif(2.f * (float)(r - rint(r)), &sn, &cs);
        table[i] = make_float2(a.amplitude * cs, a.amplitude * a.sin_sign * sn);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; i++) {
        if (where[i] < 0) continue;
        const int t = where[i] >> 16, u = where[i] & 0xffff;
        P ol = lo[i], oh = hi[i];
        if (turn[i]) {
            const float2* tp = table + t * a.pairs + V * u;
            float x[2 * V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                if constexpr (V == 1) {
                    x[0] = static_cast<float>(ol);
                    x[1] = static_cast<float>(oh);
                } else {
                    x[j] = static_cast<float>(ol[j]);
                    x[V + j] = static_cast<float>(oh[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float2 cs = tp[j];
                float& p0 = x[HALVES ? j : 2 * j];
                float& p1 = x[HALVES ? V + j : 2 * j + 1];
                const float y0 = p0 * cs.x - p1 * cs.y, y1 = p0 * cs.y + p1 * cs.x;
                p0 = y0;
                p1 = y1;
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                if constexpr (V == 1) {
                    ol = static_cast<T>(x[0]);
                    oh = static_cast<T>(x[1]);
                } else {
                    ol[j] = static_cast<T>(x[j]);
                    oh[j] = static_cast<T>(x[V + j]);
                }
            }
        }
        const int step = HALVES && u < a.rot_units ? half : V;
        *reinterpret_cast<P*>(dst[i]) = ol;
        *reinterpret_cast<P*>(dst[i] + step) = oh;
    }
}

// Turns per position of each pair: theta^(-2p / rot) / 2 pi, scaled.  False where one is not a number below
// kMaxTurns (2^31 positions of it still have 2^-2 of a turn's precision in float64).
constexpr double kMaxTurns = 1048576.;
bool make_turns(const irodori_rope_desc& d, double* turns) {
    const int n = d.rot_dim / 2;
    // Powers by products in the host's 64-bit significands, which leave float64's own rounding; products in float64 lose up
    // to 2 n 2^-53 (2.5e-6 radians at position 2^28 with 256 pairs and a theta of 1.5).
    // (Through logarithms: pow in these numbers takes 0.5 us.)
    long double log_theta = std::log2((long double)d.theta);
    if (d.scaling == IRODORI_ROPE_NTK) log_theta += d.rot_dim / (d.rot_dim - 2.0L) * std::log2((long double)d.factor);
    const long double ratio = std::exp2(-2.0L / d.rot_dim * log_theta);
    long double f = 0.159154943091895335768884L;  // 1 / 2 pi
    for (int p = 0; p < n; p++, f *= ratio) {
        double t = (double)f;
        if (d.scaling == IRODORI_ROPE_LINEAR) {
            t /= d.factor;
        } else if (d.scaling == IRODORI_ROPE_BY_PARTS) {
            const double whole = d.trained_len * (double)f;  // turns over the trained length
            const double keep = std::min(1.0, std::max(0.0, (whole - d.beta_slow) / (d.beta_fast - d.beta_slow)));
            t *= keep + (1.0 - keep) / d.factor;
        }
        if (!(t < kMaxTurns)) return false;
        turns[p] = t;
    }
    return true;
}

int check_side(const irodori_rope_desc& d, const char* name, const void* x, const void* y, int heads, int rot_heads,
               const int64_t* xs, const int64_t* ys) {
    const std::string n(name);
    IRO_REQUIRE(x && y, IRODORI_ERR_INVALID_ARG, "irodori_op_rope: " + n + " has heads but a null pointer");
    const size_t es = dtype_bytes(d.dtype);
    IRO_REQUIRE(aligned_to(x, es) && aligned_to(y, es), IRODORI_ERR_INVALID_ARG,
                "irodori_op_rope: " + n + " is not aligned to its element type");
    IRO_REQUIRE(rot_heads >= 0 && rot_heads <= heads, IRODORI_ERR_SHAPE,
                "irodori_op_rope: " + n + "_rot_heads must be between 0 and the heads");
    const int64_t dims[3] = {d.batch, d.seq, heads};
    IRO_REQUIRE(strides_readable(dims, xs), IRODORI_ERR_SHAPE, "irodori_op_rope: " + n + " has a negative or too large stride");
    IRO_REQUIRE(strides_disjoint(dims, ys, d.head_dim), IRODORI_ERR_SHAPE,
                "irodori_op_rope: the strides of " + n + "_out let its elements overlap");
    if (x == y)
        for (int i = 0; i < 3; i++)
            IRO_REQUIRE(dims[i] == 1 || xs[i] == ys[i], IRODORI_ERR_SHAPE,
                        "irodori_op_rope: " + n + " in place needs equal strides");
    return IRODORI_OK;
}

int check_rope(const irodori_rope_desc* dp) {
    IRO_REQUIRE(dp, IRODORI_ERR_INVALID_ARG, "irodori_op_rope: null description");
    const irodori_rope_desc& d = *dp;
    IRO_REQUIRE(op_dtype_ok(d.dtype), IRODORI_ERR_DTYPE, "irodori_op_rope: dtype must be F32, BF16 or F16");
    IRO_REQUIRE(d.batch > 0 && d.seq > 0 && d.head_dim > 0, IRODORI_ERR_SHAPE, "irodori_op_rope: dims must be positive");
    IRO_REQUIRE(d.q_heads >= 0 && d.k_heads >= 0 && d.q_heads <= 16384 && d.k_heads <= 16384 && d.q_heads + d.k_heads > 0,
                IRODORI_ERR_SHAPE, "irodori_op_rope: q_heads and k_heads must be in [0, 16384], one of them positive");
    IRO_REQUIRE(d.head_dim <= kMaxDim, IRODORI_ERR_SHAPE, "irodori_op_rope: head_dim must be at most 1024");
    IRO_REQUIRE(d.rot_dim >= 2 && d.rot_dim % 2 == 0 && d.rot_dim <= d.head_dim && d.rot_dim <= kMaxRot, IRODORI_ERR_SHAPE,
                "irodori_op_rope: rot_dim must be even, at least 2 and at most head_dim and 512");
    IRO_REQUIRE(d.layout == IRODORI_ROPE_INTERLEAVED || d.layout == IRODORI_ROPE_HALVES, IRODORI_ERR_CONFIG,
                "irodori_op_rope: unknown layout");
    IRO_REQUIRE(std::isfinite(d.theta) && d.theta > 0, IRODORI_ERR_CONFIG, "irodori_op_rope: theta must be positive");
    IRO_REQUIRE(std::fabs(d.amplitude) <= 1e38, IRODORI_ERR_CONFIG, "irodori_op_rope: amplitude must be at most 1e38 in magnitude");
    IRO_REQUIRE(d.scaling >= IRODORI_ROPE_UNSCALED && d.scaling <= IRODORI_ROPE_BY_PARTS, IRODORI_ERR_CONFIG,
                "irodori_op_rope: unknown scaling");
    if (d.scaling != IRODORI_ROPE_UNSCALED)
        IRO_REQUIRE(std::isfinite(d.factor) && d.factor > 0, IRODORI_ERR_CONFIG, "irodori_op_rope: factor must be positive");
    IRO_REQUIRE(d.scaling != IRODORI_ROPE_NTK || d.rot_dim > 2, IRODORI_ERR_CONFIG,
                "irodori_op_rope: the base's scaling needs rot_dim above 2");
    if (d.scaling == IRODORI_ROPE_BY_PARTS)
        IRO_REQUIRE(std::isfinite(d.trained_len) && d.trained_len > 0 && std::isfinite(d.beta_slow) &&
                        std::isfinite(d.beta_fast) && d.beta_fast > d.beta_slow,
                    IRODORI_ERR_CONFIG,
                    "irodori_op_rope: scaling by parts needs a positive trained_len and beta_fast above beta_slow");
    IRO_REQUIRE(d.seq <= 1 << 30 && d.first_pos <= INT32_MAX - d.seq, IRODORI_ERR_SHAPE,
                "irodori_op_rope: more than 2^30 tokens, or positions past 2^31");
    return IRODORI_OK;
}

unsigned ceil_inv(int d) { return (unsigned)(((1ull << 32) + d - 1) / d); }

// An output over something that is read or over the other one (q_out may be q, and k_out k).
bool outputs_overlap(const irodori_rope_desc& d, const RopeArgs& a) {
    const size_t es = dtype_bytes(d.dtype);
    const int64_t nq[3] = {d.batch, d.seq, d.q_heads}, nk[3] = {d.batch, d.seq, d.k_heads};
    auto box = [&](const void* p, const int64_t (&n)[3], const int64_t* s) { return Box(n[2] ? p : nullptr, es, n, s, d.head_dim); };
    const Box q = box(a.q.x, nq, a.q.xs), k = box(a.k.x, nk, a.k.xs), qo = box(a.q.y, nq, a.q.ys), ko = box(a.k.y, nk, a.k.ys);
    const Box pos(a.positions, (int64_t)4 * d.batch * d.seq), len(a.lengths, (int64_t)4 * d.batch);
    return (a.q.x != a.q.y && overlap(qo, q)) || (a.k.x != a.k.y && overlap(ko, k)) || overlap(qo, k) || overlap(ko, q) ||
           overlap(qo, ko) || overlap(qo, pos) || overlap(qo, len) || overlap(ko, pos) || overlap(ko, len);
}

template <typename T, int V, bool HALVES>
int launch(const irodori_rope_desc& d, RopeArgs& a, hipStream_t st) {
    const int total = a.q.heads + a.k.heads, most = 256 * kItems;
    a.rot_units = d.rot_dim / (2 * V);
    a.units = a.rot_units + (d.head_dim - d.rot_dim) / (2 * V);
    // A workgroup takes whole heads of whole tokens: as many heads as it holds, then as many tokens,
    // fewer while the launch does not fill the chip's 256 CUs four times.
    a.heads = std::min(total, most / a.units);
    a.head_blocks = (total + a.heads - 1) / a.heads;
    a.heads = (total + a.head_blocks - 1) / a.head_blocks;
    a.tokens = std::max(1, std::min({most / (a.units * a.heads), kTable / a.pairs, d.seq}));
    while (a.tokens > 1 && (int64_t)d.batch * ((d.seq + a.tokens - 1) / a.tokens) * a.head_blocks < 1024) a.tokens = (a.tokens + 1) / 2;
    a.tok_blocks = (d.seq + a.tokens - 1) / a.tokens;
    a.div_units = ceil_inv(a.units);
    a.div_heads = ceil_inv(a.heads);
    const int64_t wgs = (int64_t)d.batch * a.tok_blocks * a.head_blocks;
    IRO_REQUIRE(wgs <= UINT32_MAX / 256, IRODORI_ERR_SHAPE, "irodori_op_rope: too many tokens for one launch");
    IRO_REQUIRE(!outputs_overlap(d, a), IRODORI_ERR_INVALID_ARG, "irodori_op_rope: an output overlaps another argument");
    rope_kernel<T, V, HALVES><<<(unsigned)wgs, 256, 0, st>>>(a);
    return check_launch("rope");
}

template <typename T, int V>
int launch_layout(const irodori_rope_desc& d, RopeArgs& a, hipStream_t st) {
    return d.layout == IRODORI_ROPE_HALVES ? launch<T, V, true>(d, a, st) : launch<T, V, false>(d, a, st);
}
// The widest pack that divides both parts of a head (any alignment of the element's size will do).
template <typename T>
int launch_width(const irodori_rope_desc& d, RopeArgs& a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int rest = d.head_dim - d.rot_dim;
    if (d.rot_dim % (2 * V) == 0 && rest % (2 * V) == 0) return launch_layout<T, V>(d, a, st);
    if (d.rot_dim % V == 0 && rest % V == 0) return launch_layout<T, V / 2>(d, a, st);
    return launch_layout<T, 1>(d, a, st);
}

}  // namespace

extern "C" {

int irodori_op_rope(const irodori_rope_desc* desc, const void* q, void* q_out, const void* k, void* k_out,
                    const int32_t* positions, const int32_t* lengths, void* stream) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_rope(desc));
    const irodori_rope_desc& d = *desc;
    if (d.q_heads) IRO_TRY(check_side(d, "q", q, q_out, d.q_heads, d.q_rot_heads, d.q_strides, d.q_out_strides));
    if (d.k_heads) IRO_TRY(check_side(d, "k", k, k_out, d.k_heads, d.k_rot_heads, d.k_strides, d.k_out_strides));
    if (d.q_heads && d.k_heads)
        IRO_REQUIRE(q_out != k_out && q_out != k && k_out != q, IRODORI_ERR_INVALID_ARG,
                    "irodori_op_rope: one side's output is the other side's tensor");
    IRO_REQUIRE(d.head_dim % 2 == 0, IRODORI_ERR_SHAPE, "irodori_op_rope: head_dim must be even");
    IRO_REQUIRE(aligned_to(positions, 4) && aligned_to(lengths, 4), IRODORI_ERR_INVALID_ARG,
                "irodori_op_rope: positions or lengths are not aligned");
    RopeArgs a;
    auto side = [](const void* x, void* y, const int64_t* xs, const int64_t* ys, int heads, int rot) {
        return RopeSide{x, y, {xs[0], xs[1], xs[2]}, {ys[0], ys[1], ys[2]}, heads, rot};
    };
    a.q = side(q, q_out, d.q_strides, d.q_out_strides, d.q_heads, d.q_rot_heads);
    a.k = side(k, k_out, d.k_strides, d.k_out_strides, d.k_heads, d.k_rot_heads);
    a.positions = positions;
    a.lengths = lengths;
    a.first_pos = d.first_pos;
    a.batch = d.batch;
    a.seq = d.seq;
    a.pairs = d.rot_dim / 2;
    a.amplitude = (float)d.amplitude;
    a.sin_sign = d.inverse ? -1.f : 1.f;
    IRO_REQUIRE(make_turns(d, a.turns), IRODORI_ERR_CONFIG, "irodori_op_rope: theta and the scaling give a frequency that is too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    IRO_TRY(check_op_stream(st, "irodori_op_rope"));
    if (d.dtype == IRODORI_DTYPE_BF16) return launch_width<bf16>(d, a, st);
    if (d.dtype == IRODORI_DTYPE_F16) return launch_width<f16>(d, a, st);
    return launch_width<float>(d, a, st);
    IRO_GUARD_END
}

}  // extern "C"
