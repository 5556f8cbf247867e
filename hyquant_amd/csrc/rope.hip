// Position rotation of queries and keys with the norms of their heads, on its
// own and on the way into a paged cache of 4 or 8 bits; the 8-bit cache's
// append and read-back.
//
// A head's row x of D channels becomes
//   y = x rsqrt(mean(x^2) + eps) w                      (where there is a weight)
//   (y_a, y_b) <- (y_a c - y_b s, y_b c + y_a s)        for R / 2 channel pairs
// with c and s from row `position` of a table.  8-bit pages hold int8 codes
// [pages, key heads, page, D] and one fp32 scale, a power of two, for each block
// of 16 tokens of a page and key head.
#include "hyq_common.h"

#include <algorithm>
#include <cmath>
#include <string>

namespace hyq {
namespace {

constexpr int BLOCK = 16;                // tokens of an 8-bit scale
constexpr int64_t MOST_THREADS = (int64_t{1} << 32) - 1024;    // of a launch, along a dimension

struct Rows {                            // [batch, n, heads, D], contiguous channels
    const uint16_t* p;
    int64_t sb, sn, sh;
};
struct Pool {
    int8_t *kp, *vp;
    int64_t ps_page, ps_head;
    void *ks, *vs;                       // fp16 per token (4 bits), fp32 per block (8 bits)
    int64_t ss_page, ss_head;
    int64_t num_slots;
    const int64_t* slots;
    int32_t page_log2;
};
struct RopeArgs {
    Rows q, k, v;
    uint16_t *qo, *ko;                   // contiguous
    const void *cos, *sin;               // [batch or 1, rows, half]
    int64_t cs_b, cs_m, table_rows;
    const int64_t* positions;            // or null: token i of each batch entry has row i
    const void *qw, *kw;                 // [D] or null
    double eps;
    uint32_t tokens, n, hq, hk;          // tokens = batch * n
    int32_t half;                        // R / 2, a multiple of 8
    int32_t interleaved, table_type, weight_fp32;
    uint32_t q_blocks;                   // workgroups of the q rows in an append's grid
    Pool pool;
};

template <bool F16>
__device__ __forceinline__ float half_at(uint32_t w, int hi) {
    if constexpr (F16) return f16_bits_to_f32(static_cast<uint16_t>(hi ? w >> 16 : w));
    else return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
}
// four values (fp32: type 0, bf16: 1, fp16: 2), aligned to their size
__device__ __forceinline__ void load4(const void* p, int64_t at, int type, float (&f)[4]) {
    if (type == 0) {
        const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = type == 1 ? half_at<false>(j < 2 ? v.x : v.y, j & 1) : half_at<true>(j < 2 ? v.x : v.y, j & 1);
    }
}

// ---- over the D/8 lanes of a row (8 or 16), by DPP row operations ----
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ int dpp(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, false); }
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = dpp<CTRL>(static_cast<int>(b)), hi = dpp<CTRL>(static_cast<int>(b >> 32));
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
template <int LPT, typename T, typename OP>
__device__ __forceinline__ T over_lanes(T v, OP op) {
    v = op(v, dpp<0xb1>(v));             // quad_perm [1,0,3,2]
    v = op(v, dpp<0x4e>(v));             // quad_perm [2,3,0,1]
    v = op(v, dpp<0x141>(v));            // row_half_mirror
    if (LPT == 16) v = op(v, dpp<0x140>(v));       // row_mirror
    return v;
}
template <int LPT, typename T>
__device__ __forceinline__ T lanes_sum(T v) { return over_lanes<LPT>(v, [](T a, T b) { return a + b; }); }
template <int LPT, typename T>
__device__ __forceinline__ T lanes_max(T v) { return over_lanes<LPT>(v, [](T a, T b) { return b > a ? b : a; }); }

// 1 / sqrt(x): the hardware's estimate (2^-24) and two Newton steps, the division
// where that has no range
__device__ __forceinline__ double inv_root(double x) {
    if (!(x >= 0x1p-1000 && x < static_cast<double>(INFINITY))) return 1.0 / sqrt(x);
    double r = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = __builtin_fma(0.5 * r, __builtin_fma(-x * r, r, 1.0), r);
    return r;
}
// The mean of a row's squares and eps, in SUM
template <int D, typename SUM>
__device__ __forceinline__ SUM mean_square(const float (&x)[8], double eps) {
    SUM sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += static_cast<SUM>(x[i]) * static_cast<SUM>(x[i]);
    return lanes_sum<D / 8>(sum) * static_cast<SUM>(1.0 / D) + static_cast<SUM>(eps);
}
// The inverse root mean square of a row, by the hardware's estimate (a unit in the last place) where
// 32 bits hold the mean, from 64 bits else.  (64 bits for every row of a rotation: 232 us where this
// takes 222.)  Rows whose inverse is no normal 32-bit number are scaled on the way by a power of two
// that the inverse makes up for: subnormal rows have inverses up to 2^137.
template <int D>
__device__ __forceinline__ float inv_rms(float (&x)[8], double eps) {
    const float mean = mean_square<D, float>(x, eps);
    if (mean >= 0x1p-90f && mean <= 0x1p120f) return __builtin_amdgcn_rsqf(mean);
    const double inv = inv_root(mean_square<D, double>(x, eps));
    const float by = inv > 0x1p100 ? 0x1p32f : inv < 0x1p-100 ? 0x1p-8f : 1.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= by;
    return static_cast<float>(inv * (1.0f / by));
}

__device__ __forceinline__ uint32_t batch_of(const RopeArgs& a, uint32_t t) { return a.tokens == a.n ? 0 : t / a.n; }

// The row of the table for token t; false: its position is outside of it
__device__ __forceinline__ bool table_row(const RopeArgs& a, uint32_t t, int64_t& at) {
    if (a.positions) {
        const int64_t m = a.positions[t];
        const bool ok = static_cast<uint64_t>(m) < static_cast<uint64_t>(a.table_rows);
        at = ok ? m * a.cs_m : 0;
        return ok;
    }
    const uint32_t b = batch_of(a, t);
    at = b * a.cs_b + (t - b * a.n) * a.cs_m;
    return true;
}
__device__ __forceinline__ const uint16_t* row_of(const RopeArgs& a, const Rows& r, uint32_t t, uint32_t h) {
    const uint32_t b = batch_of(a, t);
    return r.p + b * r.sb + (t - b * a.n) * r.sn + h * r.sh;
}

// A lane's channels of a row: a .. a + 3 and b .. b + 3.  Each rotated pair is in
// one lane: no value is read or computed twice.
struct Lane {
    int a, b;
    bool turns;                          // they are rotated, by the table's columns j .. j + 3
    int j;
};
__device__ __forceinline__ Lane lane_of(const RopeArgs& args, int sub) {
    if (args.interleaved) return Lane{8 * sub, 8 * sub + 4, 4 * sub < args.half, 4 * sub};
    const int left = 4 * sub - args.half;          // (half is a multiple of 8)
    if (left < 0) return Lane{4 * sub, args.half + 4 * sub, true, 4 * sub};
    return Lane{2 * args.half + 2 * left, 2 * args.half + 2 * left + 4, false, 0};
}
// A token's angles at the lane's channels, and the weights there
struct Angles {
    float c[4], s[4];
};
__device__ __forceinline__ Angles load_angles(const RopeArgs& a, const Lane& l, int64_t at) {
    Angles k{};
    if (l.turns) {
        load4(a.cos, at + l.j, a.table_type, k.c);
        load4(a.sin, at + l.j, a.table_type, k.s);
    }
    return k;
}
struct Weights {
    float w[8];
    bool norm;
};
template <bool F16>
__device__ __forceinline__ Weights load_weights(const RopeArgs& a, const Lane& l, const void* w) {
    Weights k{};
    k.norm = w != nullptr;
    if (w) {
        const int type = a.weight_fp32 ? 0 : F16 ? 2 : 1;
        float lo[4], hi[4];
        load4(w, l.a, type, lo);
        load4(w, l.b, type, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) { k.w[i] = lo[i]; k.w[4 + i] = hi[i]; }
    }
    return k;
}
struct Raw {
    uint2 a, b;
};
__device__ __forceinline__ Raw load_raw(const uint16_t* row, const Lane& l) {
    return Raw{*reinterpret_cast<const uint2*>(row + l.a), *reinterpret_cast<const uint2*>(row + l.b)};
}
template <bool F16>
__device__ __forceinline__ void unpack(const Raw& r, float (&x)[8]) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.b.x, r.b.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = half_at<F16>(w[i >> 1], i & 1);
}

// A lane's channels normalised and rotated, in T; the norm's sum in SUM.  `most`: where it is
// asked for, the sum of the magnitudes that each value is the sum of, 0 where it is not computed.
template <int D, typename SUM, typename T, bool MOST = false>
__device__ __forceinline__ void turn(const RopeArgs& a, const Lane& l, const Angles& k, const Weights& w, const float (&x)[8], T (&y)[8],
                                     T (*most)[8] = nullptr) {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(x[i]);
    bool rough = false;                  // the inverse root is no normal 32-bit number: the bound does not hold
    if (w.norm) {
        T inv;
        if constexpr (std::is_same_v<SUM, float>) inv = inv_rms<D>(v, a.eps);
        else inv = static_cast<T>(inv_root(mean_square<D, SUM>(x, a.eps)));
        if constexpr (MOST) rough = !(inv >= static_cast<T>(0x1p-120) && inv <= static_cast<T>(0x1p120));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * static_cast<T>(w.w[i]);
    }
    auto mag = [](T z) { return z < 0 ? -z : z; };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = v[i];
        if constexpr (MOST) (*most)[i] = w.norm ? mag(v[i]) : static_cast<T>(0);       // (a value that passes is exact)
    }
    auto pair = [&](int p, int q, T c, T s) {
        const T f = v[p], g = v[q];
        y[p] = f * c - g * s;
        y[q] = g * c + f * s;
        if constexpr (MOST) {
            (*most)[p] = mag(f * c) + mag(g * s);
            (*most)[q] = mag(g * c) + mag(f * s);
        }
    };
    if (l.turns) {
        if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pair(2 * i, 2 * i + 1, k.c[i], k.s[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) pair(i, i + 4, k.c[i], k.s[i]);
        }
    }
    if constexpr (MOST) {
        if (rough) (*most)[0] = static_cast<T>(INFINITY);
    }
}

template <bool F16>
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
    if constexpr (F16)
        return make_uint2(f32_to_f16_bits(a) | static_cast<uint32_t>(f32_to_f16_bits(b)) << 16,
                          f32_to_f16_bits(c) | static_cast<uint32_t>(f32_to_f16_bits(d)) << 16);
    else return make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}

// HP heads of a token into contiguous rows: their loads in flight together, the
// table's row and the weights loaded once.  A position outside the table gives zeros.
// Bound by bytes, 2 D in and 2 D out of a row, where there are many: four prompts of 8191
// tokens, 64 + 8 heads of 128 (1.21 GB), take 221 us, 5.5 TB/s, where a copy of
// 1 GiB reaches 5.05.  A pair in two lanes, each reading and normalising both
// values of it, took 306.  Few rows are bound by the launch: 16 tokens 3.2 us.
template <int D, bool F16, int HP>
__device__ __forceinline__ void rotate_heads(const RopeArgs& a, const Rows& src, uint16_t* dst, const void* w, uint32_t unit, uint32_t heads,
                                             int sub) {
    const uint32_t per = (heads + HP - 1) / HP, t = unit / per, h0 = (unit - t * per) * HP;
    if (t >= a.tokens) return;
    const Lane l = lane_of(a, sub);
    Raw raw[HP];
#pragma unroll
    for (int i = 0; i < HP; ++i) raw[i] = load_raw(row_of(a, src, t, min(h0 + i, heads - 1)), l);
    int64_t at;
    const bool ok = table_row(a, t, at);
    const Angles k = load_angles(a, l, at);
    const Weights wt = load_weights<F16>(a, l, w);
    uint16_t* out = dst + (static_cast<int64_t>(t) * heads + h0) * D;
#pragma unroll
    for (int i = 0; i < HP; ++i) {
        float x[8], y[8];
        unpack<F16>(raw[i], x);
        turn<D, float>(a, l, k, wt, x, y);
        if (h0 + i < heads) {
            *reinterpret_cast<uint2*>(out + i * D + l.a) = ok ? pack4<F16>(y[0], y[1], y[2], y[3]) : make_uint2(0, 0);
            *reinterpret_cast<uint2*>(out + i * D + l.b) = ok ? pack4<F16>(y[4], y[5], y[6], y[7]) : make_uint2(0, 0);
        }
    }
}

template <int D, bool F16, int HP>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
    constexpr int LPT = D / 8;
    const int sub = threadIdx.x & (LPT - 1);
    const uint32_t at = threadIdx.x / LPT;
    if (blockIdx.x < a.q_blocks) rotate_heads<D, F16, HP>(a, a.q, a.qo, a.qw, blockIdx.x * (256 / LPT) + at, a.hq, sub);
    else rotate_heads<D, F16, HP>(a, a.k, a.ko, a.kw, (blockIdx.x - a.q_blocks) * (256 / LPT) + at, a.hk, sub);
}

// ---- codes of rotated keys ----
// They are those of the formula: a key is rotated in 32 bits (the norm's sum in 64),
// and again in 64 bits where 32 bits' error may reach over a code's or a scale's
// border (a wavefront decides for its rows; one of 55 to 95 does, of Gaussian keys).  The error of
// a value is at most 5 2^-24 of the magnitudes that it is the sum of: the inverse
// root's rounding, two products, and the rotation's product and sum.
constexpr float TURN_ERROR = 6.0f * 0x1p-24f;

// The correctly rounded quotient x / s (s > 0 finite) from inv = RN(1 / s)
__device__ __forceinline__ double quot_rn(double x, double s, double inv) {
    const double q = x * inv;
    return __builtin_fma(__builtin_fma(-q, s, x), inv, q);
}

// 4 bits: scale = fp16(fp32(max(amax, 1e-5) / 7)), code = RNE(x / scale)
template <int D, bool F16>
__device__ __forceinline__ void key_codes4(const RopeArgs& a, const Lane& l, const Angles& k, const Weights& wt, const Raw& raw, _Float16& s16, int (&c)[8]) {
    float x[8], y[8], err[8];
    unpack<F16>(raw, x);
    turn<D, double, float, true>(a, l, k, wt, x, y, &err);
    float amax = 0.f, off = 0.f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        err[i] *= TURN_ERROR;
        amax = fmaxf(amax, fabsf(y[i]));
        off = fmaxf(off, err[i]);
        fine = fine && y[i] == y[i];
    }
    amax = lanes_max<D / 8>(amax);
    off = lanes_max<D / 8>(off) + amax * 0x1p-22f;
    s16 = static_cast<_Float16>(fmaxf(amax, 1e-5f) * (1.0f / 7.0f));
    const float sf = static_cast<float>(s16), inv = 1.0f / sf;
    fine = fine && sf <= 65504.0f && static_cast<_Float16>(fmaxf(amax - off, 1e-5f) * (1.0f / 7.0f)) == s16 &&
           static_cast<_Float16>(fmaxf(amax + off, 1e-5f) * (1.0f / 7.0f)) == s16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = y[i] * inv, z = rintf(q);
        // (2^-19: the quotient's own error, at most 8 of three roundings)
        fine = fine && fabsf(q - z) + err[i] * inv < 0.5f - 0x1p-19f;
        c[i] = static_cast<int>(fminf(fmaxf(z, -8.0f), 7.0f));
    }
    if (__builtin_amdgcn_ballot_w64(!fine)) {
        double v[8], top = 0.0;
        turn<D, double>(a, l, k, wt, x, v);
        int nan = 0;                     // (a maximum passes them over)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top = fmax(top, fabs(v[i]));
            nan |= v[i] != v[i];
        }
        top = lanes_max<D / 8>(nan) ? __builtin_nan("") : fmax(lanes_max<D / 8>(top), 1e-5);
        s16 = static_cast<_Float16>(static_cast<float>(top / 7.0));
        const double sd = static_cast<double>(s16), invd = 1.0 / sd;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double q = sd <= 65504.0 ? quot_rn(v[i], sd, invd) : v[i] / sd;
            c[i] = static_cast<int>(fmin(fmax(rint(q), -8.0), 7.0));
        }
    }
}

// q's heads, and a K and a V row of a token and head each, in one launch.  Bound by
// bytes for many rows: 8191 tokens of 64 + 2 x 8 heads of 128 (311 MB) take 71 us,
// 4.4 TB/s (with every key in 64 bits 127); 48 decode steps 4.4 us, the
// launch and slot -> page -> row.
template <int D, bool F16, int HP>
__global__ __launch_bounds__(256) void paged_rope_append_kernel(RopeArgs a) {
    constexpr int LPT = D / 8;
    const int sub = threadIdx.x & (LPT - 1);
    const uint32_t unit = threadIdx.x / LPT;
    if (blockIdx.x < a.q_blocks) {
        rotate_heads<D, F16, HP>(a, a.q, a.qo, a.qw, blockIdx.x * (256 / LPT) + unit, a.hq, sub);
        return;
    }
    const uint32_t row = (blockIdx.x - a.q_blocks) * (256 / LPT) + unit, t = row / a.hk, h = row - t * a.hk;
    if (t >= a.tokens) return;
    const Lane l = lane_of(a, sub);
    const Raw kr = load_raw(row_of(a, a.k, t, h), l);
    const uint4 vr = reinterpret_cast<const uint4*>(row_of(a, a.v, t, h))[sub];
    const int64_t slot = a.pool.slots[t];
    int64_t at;
    const bool ok = table_row(a, t, at);
    const Angles k = load_angles(a, l, at);
    const Weights wt = load_weights<F16>(a, l, a.kw);
    float x[8], amax = 0.f;
    const uint32_t w[4] = {vr.x, vr.y, vr.z, vr.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = half_at<F16>(w[i >> 1], i & 1);
        amax = fmaxf(amax, fabsf(x[i]));
    }
    _Float16 ks, vs;
    uint32_t cv[8];
    int ck[8];
    quant_row_codes<4>(x, fmaxf(lanes_max<LPT>(amax), 1e-5f), vs, cv);
    key_codes4<D, F16>(a, l, k, wt, kr, ks, ck);
    if (!ok || slot < 0 || slot >= a.pool.num_slots) return;
    uint32_t vw = 0, ka = 0, kb = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) vw |= (cv[i] & 15u) << (4 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ka |= (static_cast<uint32_t>(ck[i]) & 15u) << (4 * i);
        kb |= (static_cast<uint32_t>(ck[4 + i]) & 15u) << (4 * i);
    }
    const int64_t page = slot >> a.pool.page_log2, off = slot & ((1 << a.pool.page_log2) - 1);
    const int64_t to = page * a.pool.ps_page + h * a.pool.ps_head + off * (D / 2);
    reinterpret_cast<uint32_t*>(a.pool.vp + to)[sub] = vw;
    *reinterpret_cast<uint16_t*>(a.pool.kp + to + l.a / 2) = static_cast<uint16_t>(ka);
    *reinterpret_cast<uint16_t*>(a.pool.kp + to + l.b / 2) = static_cast<uint16_t>(kb);
    if (sub == 0) {
        const int64_t so = page * a.pool.ss_page + h * a.pool.ss_head + off;
        static_cast<uint16_t*>(a.pool.ks)[so] = __builtin_bit_cast(uint16_t, ks);
        static_cast<uint16_t*>(a.pool.vs)[so] = __builtin_bit_cast(uint16_t, vs);
    }
}

// ---------------------------------------------------------------------------
// 8-bit pages
// ---------------------------------------------------------------------------
// The exponent of a block's scale: the smallest e with max(amax, 1e-5) <= 127
// 2^e, so that x 2^-e and its rounding are exact and so are codes that are
// rounded again for a larger e.  Values past 127 2^MOST_E (and what is not
// finite) make the block's scale NaN.
constexpr int AGAIN = 8;                 // kept rows that are rounded again at a time: two rounds of loads for the 15 there may be (200 decode steps 8.1 us, with 5 8.3: as much as launches of one kernel differ)
constexpr int SKIP = 8;                  // slots a lane looks at together in a stretch without any
constexpr int LEAST_E = -23;             // of 1e-5
constexpr int MOST_E = 40, BAD_E = 1 << 20, NO_E = -(1 << 20);
__device__ __forceinline__ int exponent(double amax) {
    if (!(amax <= 127.0 * 0x1p40)) return BAD_E;
    const uint64_t b = __builtin_bit_cast(uint64_t, fmax(amax, 1e-5));
    return static_cast<int>((b >> 52) & 2047) - 1022 - 7 + ((b & 0xfffffffffffffull) > 0xfc00000000000ull ? 1 : 0);
}
__device__ __forceinline__ int exponent(float amax) {                    // (1e-5 and its fp32 neighbour have the same)
    if (!(amax <= 127.0f * 0x1p40f)) return BAD_E;
    const uint32_t b = __float_as_uint(fmaxf(amax, 1e-5f));
    return static_cast<int>(b >> 23) - 126 - 7 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// A run of tokens whose slots lie in one block is worked on by the workgroup that
// has its first token among its 16, K and V of one head: the block's scale is the
// largest that its new rows, and the rows before them, need; rows before the
// run's first live one (a token whose position is outside the table is not) stay,
// and are rounded again where the scale has grown.  The rows of a long run that
// starts at the window's token f are the tokens f .. f + 15: the lanes of the first f
// rows take those behind the window.  Only where more runs start in it may a second pass
// be left.  Tokens whose slot is outside the pool belong to no run and part none:
// runs that they parted would be two workgroups' on one block.  60 chunks of 33 to
// 1501 tokens, 32 + 2 x 8 heads of 64 (284 MB with q), take 73 us, 3.9 TB/s: q's rows
// alone 45; VALU issue is half of it, a workgroup's chain slots -> rows and scales ->
// exponents -> codes the rest.  Windows that are worked on row by row twice (16 tokens
// and the 16 behind them), K and V apart: 146.  200 decode steps 8 us, the chain, and
// codes again where a scale grows.
template <int D, bool F16, bool ROPE, int HP>
__global__ __launch_bounds__(2 * D, 4) void paged8_append_kernel(RopeArgs a) {
    constexpr int LPT = D / 8;
    const int sub = threadIdx.x & (LPT - 1), r0 = threadIdx.x / LPT, lane = threadIdx.x & 63;
    if constexpr (ROPE) {
        if (blockIdx.x < a.q_blocks) {
            rotate_heads<D, F16, HP>(a, a.q, a.qo, a.qw, blockIdx.x * 16 + r0, a.hq, sub);
            return;
        }
    }
    __shared__ int need[2][32];
    const uint32_t i = blockIdx.x - a.q_blocks, win = i / a.hk, h = i - win * a.hk, t0 = win * 16;

    for (int j = threadIdx.x; j < 64; j += 2 * D) need[j >> 5][j & 31] = NO_E;
    // ---- the runs: lane l of each wavefront looks at token t0 - 1 + l, up to t0 + 31 ----
    uint32_t tok = min(max(t0 + lane, 1u) - 1, a.tokens - 1);
    auto slot_of = [&](uint32_t t) -> int64_t {
        const int64_t s = a.pool.slots[t];
        return s >= 0 && s < a.pool.num_slots ? s : -1;
    };
    int own = 16;                        // places of the window's own tokens
    int64_t slot = -1;
    const bool in = lane <= 32 && t0 + lane >= 1 && t0 + lane <= a.tokens;
    if (in) slot = slot_of(tok);
    const bool gaps = __builtin_amdgcn_ballot_w64(in && slot < 0);       // (the same in all wavefronts)
    if (gaps) {
        // Tokens without a slot do not part a run: the lanes take the tokens that have
        // one instead, the last before t0 and 32 from it on, however far apart: 4000
        // tokens without any beside 5 cost nothing that shows, 100000 0.2 ms.  (The whole
        // workgroup's search takes 50 us there, and its code costs 1.3 to 3 of the 92 us
        // of the 60 chunks.)
        uint64_t m = __builtin_amdgcn_ballot_w64(slot >= 0) & 0x1fffeu;
        if (!m) return;
        own = __builtin_popcountll(m);
        int64_t before = -1;
        const int64_t first = __shfl(slot, __builtin_ctzll(m), 64), last = __shfl(slot, 63 - __builtin_clzll(m), 64);
        if (first & (BLOCK - 1)) {       // (a block's first row starts a run)
            for (int64_t t = static_cast<int64_t>(t0) - 1 - lane; t + lane >= 0 && before < 0; t -= 64 * SKIP) {
                int64_t s[SKIP];
#pragma unroll
                for (int j = 0; j < SKIP; ++j) s[j] = t - 64 * j >= 0 ? slot_of(static_cast<uint32_t>(t - 64 * j)) : -1;
#pragma unroll
                for (int j = 0; j < SKIP; ++j) {
                    m = __builtin_amdgcn_ballot_w64(s[j] >= 0);
                    if (m && before < 0) before = __shfl(s[j], __builtin_ctzll(m), 64);
                }
            }
        }
        slot = lane == 0 ? before : -1;
        tok = t0;
        int n = 0;                       // places taken
        bool more = true;                // the last of the window's own runs may go on
        for (int64_t t = t0; more && n < 32 && t < a.tokens; t += 64) {
            if (n >= own) {              // what is between may be long
                while (t < a.tokens) {
                    int64_t any = -1;    // (not negative where one of them has a slot)
#pragma unroll
                    for (int j = 0; j < SKIP; ++j) {
                        const int64_t at = t + 64 * j + lane;
                        any &= at < a.tokens ? slot_of(static_cast<uint32_t>(at)) : -1;
                    }
                    if (__builtin_amdgcn_ballot_w64(any >= 0)) break;
                    t += 64 * SKIP;
                }
            }
            const int64_t at = t + lane, s = at < a.tokens ? slot_of(static_cast<uint32_t>(at)) : -1;
            m = __builtin_amdgcn_ballot_w64(s >= 0);
            const int place = 1 + n + __builtin_popcountll(m & ((uint64_t{1} << lane) - 1));
            const int to = 4 * (s >= 0 && place <= 32 ? place : 63);     // (lane 63 takes no part)
            const uint32_t lo = __builtin_amdgcn_ds_permute(to, static_cast<int>(s)), hi = __builtin_amdgcn_ds_permute(to, static_cast<int>(s >> 32));
            const uint32_t who = __builtin_amdgcn_ds_permute(to, static_cast<int>(at));
            const int until = min(n + __builtin_popcountll(m), 32);
            if (lane > n && lane <= until) {
                slot = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
                tok = who;
            }
            n = until;
            const bool other = s >= 0 && at >= t0 + 16u && (s >> 4) != (last >> 4);
            more = !__builtin_amdgcn_ballot_w64(other || (s >= 0 && (s >> 4) == (last >> 4) && (s & (BLOCK - 1)) == BLOCK - 1));
        }
    }
    bool ok = true;
    if constexpr (ROPE) {
        int64_t unused;
        if (slot >= 0) ok = table_row(a, tok, unused);
    }
    const int64_t block = slot >> 4, ahead = __shfl_up(block, 1, 64);
    const uint32_t starts = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(block != ahead) >> 1);
    const uint32_t live = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok && slot >= 0) >> 1);
    if (!(starts & ((1u << own) - 1))) return;                           // (all tokens belong to a run that started before)
    const int f = __builtin_ctz(starts), end = starts >> own ? own + __builtin_ctz(starts >> own) : 32;
    const bool twice = end > 16 + f;

    struct Row {
        int r;                           // its place (where no token is without a slot, the token behind t0)
        uint32_t t;                      // its token
        bool active;
        uint32_t mine;                   // its run's live tokens
        int64_t slot;
    };
    auto row_at = [&](int p) {
        Row w;
        w.r = r0 + 16 * (p ? r0 >= f : r0 < f);
        const bool out = w.r >= end || w.r < f || (p && r0 < f);
        const uint32_t upto = starts & (0xffffffffu >> (31 - w.r));
        const int run = upto ? 31 - __builtin_clz(upto) : 0;
        const uint32_t more = run < 31 ? starts & (0xfffffffeu << run) : 0;
        w.mine = live & (0xffffffffu << run) & (more ? (1u << __builtin_ctz(more)) - 1u : 0xffffffffu);
        w.active = !out && (w.mine >> w.r) & 1;
        w.slot = __shfl(slot, w.r + 1, 64);
        w.t = gaps ? __shfl(tok, w.r + 1, 64) : min(t0 + w.r, a.tokens - 1);
        return w;
    };
    const Lane plain{8 * sub, 8 * sub + 4, false, 0}, l = ROPE ? lane_of(a, sub) : plain;
    const Weights wt = load_weights<F16>(a, l, ROPE ? a.kw : nullptr);
    Raw kr, vr;
    Angles k{};
    auto load = [&](const Row& w) {
        kr = load_raw(row_of(a, a.k, w.t, h), l);
        vr = load_raw(row_of(a, a.v, w.t, h), plain);
        if constexpr (ROPE) {
            int64_t at;
            table_row(a, w.t, at);
            k = load_angles(a, l, at);
        }
    };
    // the row's largest magnitude's bits (those of what is not finite are above all others)
    auto largest = [&](const float (&y)[8]) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(fabsf(y[j])));
        return static_cast<uint32_t>(lanes_max<LPT>(static_cast<int>(m)));
    };
    float y[8], off = 0.f;               // K's values, and how far off they may be
    auto measure = [&](const Row& w) {
        float x[8];
        unpack<F16>(kr, x);
        int e;
        if constexpr (ROPE) {
            float most[8];
            turn<D, double, float, true>(a, l, k, wt, x, y, &most);
            off = fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), fmaxf(fmaxf(most[4], most[5]), fmaxf(most[6], most[7]))) * TURN_ERROR;
            // the row's largest may be another value's than the formula's, but not its exponent
            const float amax = __uint_as_float(largest(y));
            if (!(amax < INFINITY)) off = INFINITY;        // (32 bits do not hold them)
            const float far = lanes_max<LPT>(off) + amax * 0x1p-22f;
            e = exponent(amax + far);
            if (__builtin_amdgcn_ballot_w64(w.active && !(e == LEAST_E || amax - far > 63.5f * pow2(min(e, 0x60))))) {
                double v[8], top = 0.0;
                bool good = true;
                turn<D, double>(a, l, k, wt, x, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    good = good && fabs(v[j]) <= 127.0 * 0x1p40;
                    top = fmax(top, fabs(v[j]));
                }
                e = lanes_max<LPT>(good ? exponent(top) : BAD_E);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = x[j];
            e = exponent(__uint_as_float(largest(y)));
        }
        unpack<F16>(vr, x);
        const int ev = exponent(__uint_as_float(largest(x)));
        if (sub == 0 && w.active) {      // (the order does not matter)
            atomicMax(&need[0][__builtin_ctz(w.mine)], e);
            atomicMax(&need[1][__builtin_ctz(w.mine)], ev);
        }
    };

    const int64_t hp = h * a.pool.ps_head, hs = h * a.pool.ss_head;
    struct Place {
        int64_t rows, scale;             // of the block, from the pools' first
        int first, kept;
        float old[2];
    };
    auto place = [&](const Row& w) {
        Place q;
        const int64_t s = w.active ? w.slot : 0, page = s >> a.pool.page_log2;
        const int32_t off = static_cast<int32_t>(s & ((1 << a.pool.page_log2) - 1)) & ~(BLOCK - 1);
        q.first = w.active ? __builtin_ctz(w.mine) : 0;
        q.rows = page * a.pool.ps_page + hp + off * D;
        q.scale = page * a.pool.ss_page + hs + off / BLOCK;
        const int kept = static_cast<int>(__shfl(slot, q.first + 1, 64)) & (BLOCK - 1);
        q.kept = w.active ? kept : 0;
        q.old[0] = q.kept ? static_cast<const float*>(a.pool.ks)[q.scale] : 0.f;
        q.old[1] = q.kept ? static_cast<const float*>(a.pool.vs)[q.scale] : 0.f;
        return q;
    };
    auto write = [&](const Row& w, const Place& q) {
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const float old = q.old[kind];
            int e = need[kind][q.first];
            if (q.kept) {
                if (!(old >= 0.f && old <= pow2(MOST_E + 1))) e = BAD_E;
                else if (old > 0.f) {    // the smallest power of two from it on
                    const uint32_t b = __float_as_uint(old);
                    e = max(e, static_cast<int>(b >> 23) - 127 + (b & 0x7fffffu ? 1 : 0));
                }
            }
            const bool bad = e > MOST_E + 1;
            e = max(e, -126);            // (an inactive row's)
            const float now = bad ? __builtin_nanf("") : pow2(e), inv = bad ? 0.f : pow2(-e);
            float x[8];
            if (kind == 1) unpack<F16>(vr, x);
            // x / scale + 1.5 2^23, rounded once: the code is its low byte
            uint32_t c[8];
            float edge = 0.f;            // the nearest to a code's border
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = kind ? x[j] : y[j], z = __builtin_fmaf(v, inv, 12582912.0f);
                if (ROPE && kind == 0) edge = fmaxf(edge, fabsf(__builtin_fmaf(v, inv, 12582912.0f - z)));
                c[j] = __float_as_uint(z);
            }
            if (ROPE && kind == 0) {
                if (__builtin_amdgcn_ballot_w64(w.active && !bad && off != 0.f && !(edge + off * inv < 0.5f - 0x1p-23f))) {
                    double v[8];
                    unpack<F16>(kr, x);
                    turn<D, double>(a, l, k, wt, x, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) c[j] = static_cast<uint32_t>(static_cast<int>(rint(v[j] * static_cast<double>(inv))));
                }
            }
            if (!w.active) continue;
            auto word = [&](int j) {     // the low bytes of four
                return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[j + 3], c[j + 2], 0x0c0c0400u), __builtin_amdgcn_perm(c[j + 1], c[j], 0x0c0c0400u), 0x05040100u);
            };
            int8_t* const rows = (kind ? a.pool.vp : a.pool.kp) + q.rows;
            int8_t* const row = rows + (w.slot & (BLOCK - 1)) * D;
            *reinterpret_cast<uint32_t*>(row + (kind ? plain.a : l.a)) = word(0);
            *reinterpret_cast<uint32_t*>(row + (kind ? plain.b : l.b)) = word(4);
            if (w.r != q.first) continue;
            if (q.kept && !bad && now != old) {              // (a block whose scale is NaN keeps its codes: the old scale brings them back)
                const float by = old * inv;
                uint2* const to = reinterpret_cast<uint2*>(rows) + sub;
                for (int j0 = 0; j0 < q.kept; j0 += AGAIN) {             // (AGAIN rows' loads in flight)
                    uint2 v[AGAIN];
#pragma unroll
                    for (int j = 0; j < AGAIN; ++j) v[j] = to[min(j0 + j, q.kept - 1) * LPT];
#pragma unroll
                    for (int j = 0; j < AGAIN; ++j) {
                        const uint32_t in[2] = {v[j].x, v[j].y};
                        uint32_t out[2] = {0, 0};
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            const int code = static_cast<int8_t>(in[n >> 2] >> (8 * (n & 3)));
                            out[n >> 2] |= (static_cast<uint32_t>(static_cast<int>(rintf(static_cast<float>(code) * by))) & 255u) << (8 * (n & 3));
                        }
                        if (j0 + j < q.kept) to[(j0 + j) * LPT] = make_uint2(out[0], out[1]);
                    }
                }
            }
            if (sub == 0) static_cast<float*>(kind ? a.pool.vs : a.pool.ks)[q.scale] = now;
        }
    };

    Row w = row_at(0);
    load(w);
    Place q = place(w);
    __syncthreads();                     // (need is set)
    measure(w);
    if (twice) {                         // (the same in all lanes)
        const Place q0 = q;
        w = row_at(1);
        load(w);
        q = place(w);
        measure(w);
        __syncthreads();
        write(w, q);
        w = row_at(0);
        load(w);
        measure(w);                      // (its values again: the exponents are the same)
        write(w, q0);
    } else {
        __syncthreads();
        write(w, q);
    }
}

// Rows of the cache by slot as bf16 or fp16 values, code * scale rounded once
// (exact for bf16); slots outside the pool give zero rows.  HBM-bound: 25000 tokens of 2 x 8
// heads of 64 (78 MB) take 15 us, 5.2 TB/s.
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged8_gather_kernel(Pool pool, uint16_t* ok, uint16_t* ov, uint32_t rows, uint32_t heads) {
    constexpr int LPT = D / 8;
    const int sub = threadIdx.x & (LPT - 1);
    const uint32_t row = blockIdx.x * (256 / LPT) + threadIdx.x / LPT;
    if (row >= rows) return;
    const bool is_v = blockIdx.y != 0;
    const uint32_t t = row / heads, h = row - t * heads;
    const int64_t slot = pool.slots[t];
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= 0 && slot < pool.num_slots) {
        const int64_t page = slot >> pool.page_log2;
        const int32_t off = static_cast<int32_t>(slot & ((1 << pool.page_log2) - 1));
        const uint2 w = reinterpret_cast<const uint2*>((is_v ? pool.vp : pool.kp) + page * pool.ps_page + h * pool.ps_head + off * D)[sub];
        const float s = static_cast<const float*>(is_v ? pool.vs : pool.ks)[page * pool.ss_page + h * pool.ss_head + off / BLOCK];
        const uint32_t in[2] = {w.x, w.y};
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = static_cast<float>(static_cast<int8_t>(in[i >> 2] >> (8 * (i & 3)))) * s;
    }
    const uint2 lo = pack4<F16>(y[0], y[1], y[2], y[3]), hi = pack4<F16>(y[4], y[5], y[6], y[7]);
    reinterpret_cast<uint4*>((is_v ? ov : ok) + static_cast<int64_t>(row) * D)[sub] = make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int log2i(int x) {
    int l = 0;
    while ((1 << l) < x) ++l;
    return l;
}
bool rows16(const void* p, int64_t a, int64_t b, int64_t c) { return aligned(p, 16) && (a | b | c) % 8 == 0; }

// What the calls share: heads, rows, norms and the table.  `cache`: keys are not
// stored as rows.
int check_rope(const std::string& w, const hyq_rope_params* p, bool cache) {
    if (!p) return fail(HYQ_EINVAL, w + "null parameters");
    if (p->head_dim != 64 && p->head_dim != 128) return fail(HYQ_ENOTSUP, w + "head_dim must be 64 or 128, got " + std::to_string(p->head_dim));
    if (p->batch < 0 || p->n < 0 || p->q_heads < 0 || p->k_heads < 0) return fail(HYQ_EINVAL, w + "negative size");
    if (p->q_heads > 65535 || p->k_heads > 65535) return fail(HYQ_ENOTSUP, w + "more than 65535 heads");
    if (p->dtype_fp16 != 0 && p->dtype_fp16 != 1) return fail(HYQ_EINVAL, w + "dtype_fp16 must be 0 or 1");
    if (p->rotary < 0 || p->rotary % 16 || p->rotary > p->head_dim)
        return fail(HYQ_ENOTSUP, w + "rotary must be a multiple of 16 up to head_dim, got " + std::to_string(p->rotary));
    if (p->table_type < 0 || p->table_type > 2 || (p->weight_fp32 | 1) != 1 || (p->interleaved | 1) != 1) return fail(HYQ_EINVAL, w + "bad type or order");
    if (!(p->eps >= 0.0) || std::isinf(p->eps)) return fail(HYQ_EINVAL, w + "eps must be finite and >= 0");
    // (batch and n apart: their product may pass 64 bits; an append has up to four rows' threads for a key head)
    const int64_t rows = MOST_THREADS / (p->head_dim / 8), heads = std::max(p->q_heads + (cache ? 4 : 1) * p->k_heads, 1);
    const int64_t most = rows / heads - 32;
    if (p->n > rows || p->batch > rows || (p->n && p->batch > rows / p->n) || p->batch * p->n > most)
        return fail(HYQ_ENOTSUP, w + "more than " + std::to_string(most) + " tokens of " + std::to_string(p->q_heads) + " + " + std::to_string(p->k_heads) + " heads");
    if (p->batch == 0 || p->n == 0) return HYQ_OK;
    if (p->q_heads && (!p->q || !p->q_out)) return fail(HYQ_EINVAL, w + "null q");
    if (p->k_heads && (!p->k || (!cache && !p->k_out))) return fail(HYQ_EINVAL, w + "null k");
    if (!rows16(p->q, p->q_stride_b, p->q_stride_n, p->q_stride_h) || !rows16(p->k, p->k_stride_b, p->k_stride_n, p->k_stride_h) ||
        !aligned(p->q_out, 16) || !aligned(p->k_out, 16))
        return fail(HYQ_EINVAL, w + "rows must be 16-byte aligned with strides divisible by 8");
    if (!aligned(p->q_weight, 16) || !aligned(p->k_weight, 16) || !aligned(p->positions, 8)) return fail(HYQ_EINVAL, w + "weights or positions misaligned");
    if (p->table_rows < 0) return fail(HYQ_EINVAL, w + "negative size");
    if (p->table_rows == 0 || (!p->positions && p->table_rows < p->n)) return fail(HYQ_EINVAL, w + "the table has fewer rows than there are tokens");
    if (p->rotary && (!p->cos || !p->sin)) return fail(HYQ_EINVAL, w + "null table");
    if (!aligned(p->cos, 16) || !aligned(p->sin, 16) || (p->table_stride_b | p->table_stride_m) % 8)
        return fail(HYQ_EINVAL, w + "tables must be 16-byte aligned with strides divisible by 8");
    return HYQ_OK;
}

RopeArgs args_of(const hyq_rope_params& p) {
    RopeArgs a{};
    a.q = Rows{static_cast<const uint16_t*>(p.q), p.q_stride_b, p.q_stride_n, p.q_stride_h};
    a.k = Rows{static_cast<const uint16_t*>(p.k), p.k_stride_b, p.k_stride_n, p.k_stride_h};
    a.qo = static_cast<uint16_t*>(p.q_out);
    a.ko = static_cast<uint16_t*>(p.k_out);
    a.cos = p.cos;
    a.sin = p.sin;
    a.cs_b = p.table_stride_b;
    a.cs_m = p.table_stride_m;
    a.table_rows = p.table_rows;
    a.positions = p.positions;
    a.qw = p.q_weight;
    a.kw = p.k_weight;
    a.eps = p.eps;
    a.tokens = static_cast<uint32_t>(p.batch * p.n);
    a.n = static_cast<uint32_t>(p.n);
    a.hq = static_cast<uint32_t>(p.q_heads);
    a.hk = static_cast<uint32_t>(p.k_heads);
    a.half = p.rotary / 2;
    a.interleaved = p.interleaved;
    a.table_type = p.table_type;
    a.weight_fp32 = p.weight_fp32;
    return a;
}

// A pool of `bits` bits; the slots of `tokens` tokens
int check_pool(const std::string& w, const hyq_paged_pool* p, int bits, int32_t head_dim) {
    if (!p) return fail(HYQ_EINVAL, w + "null pool");
    if (head_dim != 64 && head_dim != 128) return fail(HYQ_ENOTSUP, w + "head_dim must be 64 or 128, got " + std::to_string(head_dim));
    if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
        return fail(HYQ_ENOTSUP, w + "page_size must be a power of two from 16 to 256, got " + std::to_string(p->page_size));
    if (p->num_pages < 0 || p->num_pages > (int64_t{1} << 30)) return fail(HYQ_EINVAL, w + "num_pages out of range");
    if (p->num_pages == 0) return HYQ_OK;
    if (!p->k_pages || !p->v_pages || !p->k_scale || !p->v_scale) return fail(HYQ_EINVAL, w + "null cache pointer");
    if (!aligned(p->k_pages, 16) || !aligned(p->v_pages, 16) || p->p_stride_page % 16 || p->p_stride_head % 16)
        return fail(HYQ_EINVAL, w + "code pages must be 16-byte aligned with strides divisible by 16");
    const size_t size = bits == 4 ? 2 : 4;
    if (!aligned(p->k_scale, size) || !aligned(p->v_scale, size)) return fail(HYQ_EINVAL, w + "scales misaligned");
    return HYQ_OK;
}
Pool pool_of(const hyq_paged_pool& p, const int64_t* slots) {
    return Pool{p.k_pages, p.v_pages, p.p_stride_page, p.p_stride_head, p.k_scale, p.v_scale, p.s_stride_page, p.s_stride_head,
                p.num_pages * p.page_size, slots, log2i(p.page_size)};
}

unsigned blocks_of(uint64_t rows, unsigned per) { return static_cast<unsigned>((rows + per - 1) / per); }

// Heads that a lane group takes after the other.  With one the rows of a small step
// spread over more of the chip, with four the table's row and the weights are
// loaded less often and more loads are in flight; four from one round of resident
// wavefronts (8192) on.  Rows of 40 heads of 128 in a captured graph, one and
// four (us): 64 tokens 2.8 and 4.1, 512 tokens 4.3 and 4.9, 1024 7.4 and 7.1, 4096 21.1
// and 18.3, 16384 87.4 and 71.0 (eight: 5.5, 6.3, 8.2, 16.6 and 70.8).
constexpr int MANY = 4;
bool many_heads(uint64_t rows, int head_dim) { return rows * (head_dim / 8) >= 8192 * 64; }

template <bool ROPE, int HP>
void append8(RopeArgs a, int head_dim, bool fp16, hipStream_t st) {
    a.q_blocks = ROPE ? blocks_of(static_cast<uint64_t>(a.tokens) * ((a.hq + HP - 1) / HP), 16) : 0;
    const dim3 grid(a.q_blocks + blocks_of(a.tokens, 16) * a.hk);
    if (head_dim == 128) {
        if (fp16) paged8_append_kernel<128, true, ROPE, HP><<<grid, dim3(256), 0, st>>>(a);
        else paged8_append_kernel<128, false, ROPE, HP><<<grid, dim3(256), 0, st>>>(a);
    } else {
        if (fp16) paged8_append_kernel<64, true, ROPE, HP><<<grid, dim3(128), 0, st>>>(a);
        else paged8_append_kernel<64, false, ROPE, HP><<<grid, dim3(128), 0, st>>>(a);
    }
}
template <int HP>
void append4(RopeArgs a, int head_dim, bool fp16, hipStream_t st) {
    const unsigned per = 256 / (head_dim / 8);
    a.q_blocks = blocks_of(static_cast<uint64_t>(a.tokens) * ((a.hq + HP - 1) / HP), per);
    const dim3 grid(a.q_blocks + blocks_of(static_cast<uint64_t>(a.tokens) * a.hk, per));
    if (head_dim == 128) {
        if (fp16) paged_rope_append_kernel<128, true, HP><<<grid, dim3(256), 0, st>>>(a);
        else paged_rope_append_kernel<128, false, HP><<<grid, dim3(256), 0, st>>>(a);
    } else {
        if (fp16) paged_rope_append_kernel<64, true, HP><<<grid, dim3(256), 0, st>>>(a);
        else paged_rope_append_kernel<64, false, HP><<<grid, dim3(256), 0, st>>>(a);
    }
}
template <int HP>
void rotate(RopeArgs a, int head_dim, bool fp16, hipStream_t st) {
    const unsigned per = 256 / (head_dim / 8);
    a.q_blocks = blocks_of(static_cast<uint64_t>(a.tokens) * ((a.hq + HP - 1) / HP), per);
    const dim3 grid(a.q_blocks + blocks_of(static_cast<uint64_t>(a.tokens) * ((a.hk + HP - 1) / HP), per));
    if (head_dim == 128) {
        if (fp16) qk_norm_rope_kernel<128, true, HP><<<grid, dim3(256), 0, st>>>(a);
        else qk_norm_rope_kernel<128, false, HP><<<grid, dim3(256), 0, st>>>(a);
    } else {
        if (fp16) qk_norm_rope_kernel<64, true, HP><<<grid, dim3(256), 0, st>>>(a);
        else qk_norm_rope_kernel<64, false, HP><<<grid, dim3(256), 0, st>>>(a);
    }
}

int check_rows(const std::string& w, const hyq_rope_params* p, const uint16_t* v, int64_t vt, int64_t vh, const int64_t* slots) {
    if (p->batch != 1) return fail(HYQ_EINVAL, w + "batch must be 1");
    if (p->k_heads < 1) return fail(HYQ_EINVAL, w + "key heads out of range");
    if (p->n == 0) return HYQ_OK;
    if (!v || !slots || !aligned(slots, 8)) return fail(HYQ_EINVAL, w + "v or slots null or misaligned");
    if (!rows16(v, vt, vh, 0)) return fail(HYQ_EINVAL, w + "rows must be 16-byte aligned with strides divisible by 8");
    return HYQ_OK;
}

}  // namespace
}  // namespace hyq

using namespace hyq;

extern "C" int hyq_qk_norm_rope(const hyq_rope_params* p, void* stream) {
    if (int st = check_rope("hyq_qk_norm_rope: ", p, false)) return st;
    const RopeArgs a = args_of(*p);
    if (a.tokens == 0 || a.hq + a.hk == 0) return HYQ_OK;
    if (many_heads(static_cast<uint64_t>(a.tokens) * (a.hq + a.hk), p->head_dim)) rotate<MANY>(a, p->head_dim, p->dtype_fp16, static_cast<hipStream_t>(stream));
    else rotate<1>(a, p->head_dim, p->dtype_fp16, static_cast<hipStream_t>(stream));
    return check_launch("hyq_qk_norm_rope");
}

extern "C" int hyq_paged_rope_append(const hyq_rope_params* p, const uint16_t* v, int64_t v_stride_t, int64_t v_stride_h,
                                     const int64_t* slots, const hyq_paged_pool* pool, void* stream) {
    const std::string w = "hyq_paged_rope_append: ";
    if (int st = check_rope(w, p, true)) return st;
    if (!pool || (pool->bits != 4 && pool->bits != 8)) return fail(HYQ_EINVAL, w + "a pool of 4 or 8 bits is needed");
    if (int st = check_pool(w, pool, pool->bits, p->head_dim)) return st;
    if (int st = check_rows(w, p, v, v_stride_t, v_stride_h, slots)) return st;
    RopeArgs a = args_of(*p);
    if (a.tokens == 0) return HYQ_OK;
    a.v = Rows{v, 0, v_stride_t, v_stride_h};
    a.pool = pool_of(*pool, slots);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool many = many_heads(static_cast<uint64_t>(a.tokens) * (a.hq + 2 * a.hk), p->head_dim);
    if (pool->bits == 8) {
        if (many) append8<true, MANY>(a, p->head_dim, p->dtype_fp16, st);
        else append8<true, 1>(a, p->head_dim, p->dtype_fp16, st);
    } else {
        if (many) append4<MANY>(a, p->head_dim, p->dtype_fp16, st);
        else append4<1>(a, p->head_dim, p->dtype_fp16, st);
    }
    return check_launch("hyq_paged_rope_append");
}

extern "C" int hyq_paged8_append(const uint16_t* k, int64_t k_stride_t, int64_t k_stride_h, const uint16_t* v, int64_t v_stride_t,
                                 int64_t v_stride_h, int32_t is_fp16, const int64_t* slots, int64_t num_tokens, int32_t kv_heads,
                                 int32_t head_dim, const hyq_paged_pool* pool, void* stream) {
    const std::string w = "hyq_paged8_append: ";
    if (int st = check_pool(w, pool, 8, head_dim)) return st;
    if (pool->bits != 8) return fail(HYQ_EINVAL, w + "a pool of 8 bits is needed");
    if (num_tokens < 0) return fail(HYQ_EINVAL, w + "negative size");
    if (kv_heads < 1 || kv_heads > 65535) return fail(HYQ_EINVAL, w + "key heads out of range");
    if (is_fp16 != 0 && is_fp16 != 1) return fail(HYQ_EINVAL, w + "is_fp16 must be 0 or 1");
    const int64_t most = MOST_THREADS / (head_dim / 8);
    if (num_tokens > most / (4 * kv_heads) - 32)
        return fail(HYQ_ENOTSUP, w + "more than " + std::to_string(most / (4 * kv_heads) - 32) + " tokens of " + std::to_string(kv_heads) + " heads");
    if (num_tokens == 0 || pool->num_pages == 0) return HYQ_OK;
    if (!k || !v || !slots || !aligned(slots, 8)) return fail(HYQ_EINVAL, w + "k, v or slots null or misaligned");
    if (!rows16(k, k_stride_t, k_stride_h, 0) || !rows16(v, v_stride_t, v_stride_h, 0))
        return fail(HYQ_EINVAL, w + "rows must be 16-byte aligned with strides divisible by 8");
    RopeArgs a{};
    a.k = Rows{k, 0, k_stride_t, k_stride_h};
    a.v = Rows{v, 0, v_stride_t, v_stride_h};
    a.tokens = a.n = static_cast<uint32_t>(num_tokens);
    a.hk = static_cast<uint32_t>(kv_heads);
    a.pool = pool_of(*pool, slots);
    append8<false, 1>(a, head_dim, is_fp16, static_cast<hipStream_t>(stream));
    return check_launch("hyq_paged8_append");
}

extern "C" int hyq_paged8_gather(const int64_t* slots, int64_t num_tokens, int32_t kv_heads, int32_t head_dim,
                                 const hyq_paged_pool* pool, int32_t out_fp16, uint16_t* k_out, uint16_t* v_out, void* stream) {
    const std::string w = "hyq_paged8_gather: ";
    if (int st = check_pool(w, pool, 8, head_dim)) return st;
    if (pool->bits != 8) return fail(HYQ_EINVAL, w + "a pool of 8 bits is needed");
    if (num_tokens < 0) return fail(HYQ_EINVAL, w + "negative size");
    if (kv_heads < 1 || kv_heads > 65535) return fail(HYQ_EINVAL, w + "key heads out of range");
    if (out_fp16 != 0 && out_fp16 != 1) return fail(HYQ_EINVAL, w + "out_fp16 must be 0 or 1");
    if (num_tokens == 0) return HYQ_OK;
    if (!k_out || !v_out || !slots) return fail(HYQ_EINVAL, w + "null pointer");
    if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(slots, 8)) return fail(HYQ_EINVAL, w + "misaligned pointer");
    const int64_t most = MOST_THREADS / (head_dim / 8);
    if (num_tokens > most / kv_heads) return fail(HYQ_ENOTSUP, w + "more than " + std::to_string(most) + " rows");
    const uint32_t rows = static_cast<uint32_t>(num_tokens * kv_heads), heads = static_cast<uint32_t>(kv_heads);
    const Pool a = pool_of(*pool, slots);
    const dim3 grid(blocks_of(rows, 256 / (head_dim / 8)), 2);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (head_dim == 128) {
        if (out_fp16) paged8_gather_kernel<128, true><<<grid, dim3(256), 0, st>>>(a, k_out, v_out, rows, heads);
        else paged8_gather_kernel<128, false><<<grid, dim3(256), 0, st>>>(a, k_out, v_out, rows, heads);
    } else {
        if (out_fp16) paged8_gather_kernel<64, true><<<grid, dim3(256), 0, st>>>(a, k_out, v_out, rows, heads);
        else paged8_gather_kernel<64, false><<<grid, dim3(256), 0, st>>>(a, k_out, v_out, rows, heads);
    }
    return check_launch("hyq_paged8_gather");
}
