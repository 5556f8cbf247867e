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
template <bool F16, typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, T (&x)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<T>(half_at<F16>(w[i >> 1], i & 1));
}
// `count` table or weight values (fp32: type 0, bf16: 1, fp16: 2), 4 * size aligned
template <int COUNT, typename T>
__device__ __forceinline__ void load_values(const void* p, int64_t at, int type, T (&f)[8]) {
    if (type == 0) {
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
#pragma unroll
        for (int i = 0; i < COUNT / 4; ++i) {
            const float4 v = s[i];
            f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
        }
    } else {
        const uint2* s = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int i = 0; i < COUNT / 4; ++i) {
            const uint2 v = s[i];
            const uint32_t w[2] = {v.x, v.y};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                f[4 * i + j] = type == 1 ? half_at<false>(w[j >> 1], j & 1) : half_at<true>(w[j >> 1], j & 1);
        }
    }
}

template <int LPT, typename T>
__device__ __forceinline__ T lanes_sum(T v) {
#pragma unroll
    for (int d = 1; d < LPT; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
template <int LPT, typename T>
__device__ __forceinline__ T lanes_max(T v) {
#pragma unroll
    for (int d = 1; d < LPT; d <<= 1) {
        const T o = __shfl_xor(v, d, 64);
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ float inv_root(float x) { return 1.0f / sqrtf(x); }
__device__ __forceinline__ double inv_root(double x) { return 1.0 / sqrt(x); }

// The row of the table for token t; false: its position is outside of it
__device__ __forceinline__ bool table_row(const RopeArgs& a, uint32_t t, int64_t& at) {
    if (a.positions) {
        const int64_t m = a.positions[t];
        at = m * a.cs_m;
        return static_cast<uint64_t>(m) < static_cast<uint64_t>(a.table_rows);
    }
    const uint32_t b = t / a.n;
    at = b * a.cs_b + (t - b * a.n) * a.cs_m;
    return true;
}
__device__ __forceinline__ const uint16_t* row_of(const RopeArgs& a, const Rows& r, uint32_t t, uint32_t h) {
    const uint32_t b = t / a.n;
    return r.p + b * r.sb + (t - b * a.n) * r.sn + h * r.sh;
}

// Channels 8 sub .. of a row, normalised and rotated, in T.  All lanes of the
// row take part.
template <int D, bool F16, typename T>
__device__ __forceinline__ void turn(const RopeArgs& a, const uint16_t* row, const void* w, int64_t at, int sub, T (&y)[8]) {
    constexpr int LPT = D / 8;
    const int lo = a.half >> 3;          // 8-channel chunks of a half
    const bool apart = !a.interleaved;
    const int other = !apart || sub >= 2 * lo ? sub : sub < lo ? sub + lo : sub - lo;     // the partners' chunk
    T x[8], p[8];
    unpack8<F16>(reinterpret_cast<const uint4*>(row)[sub], x);
    unpack8<F16>(reinterpret_cast<const uint4*>(row)[other], p);
    if (w) {
        T sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
        const T inv = inv_root(lanes_sum<LPT>(sum) * static_cast<T>(1.0 / D) + static_cast<T>(a.eps));
        const int type = a.weight_fp32 ? 0 : F16 ? 2 : 1;
        T wx[8], wp[8];
        load_values<8>(w, 8 * sub, type, wx);
        load_values<8>(w, 8 * other, type, wp);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = x[i] * inv * wx[i];
            p[i] = p[i] * inv * wp[i];
        }
    }
    if (sub >= 2 * lo) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i];
        return;
    }
    T c[8], s[8];
    if (apart) {
        const int j = 8 * (sub < lo ? sub : sub - lo);
        load_values<8>(a.cos, at + j, a.table_type, c);
        load_values<8>(a.sin, at + j, a.table_type, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i] * c[i] + (sub < lo ? -p[i] : p[i]) * s[i];
    } else {
        load_values<4>(a.cos, at + 4 * sub, a.table_type, c);
        load_values<4>(a.sin, at + 4 * sub, a.table_type, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[2 * i] = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
            y[2 * i + 1] = x[2 * i + 1] * c[i] + x[2 * i] * s[i];
        }
    }
}

template <bool F16>
__device__ __forceinline__ uint4 pack8(const float (&y)[8]) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = F16 ? f32_to_f16_bits(y[2 * i]) | (static_cast<uint32_t>(f32_to_f16_bits(y[2 * i + 1])) << 16)
                   : pack_bf16x2(y[2 * i], y[2 * i + 1]);
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// Row `row` of `heads` heads a token into contiguous rows; a position outside the
// table gives zeros.
template <int D, bool F16>
__device__ __forceinline__ void rotate_row(const RopeArgs& a, const Rows& src, uint16_t* dst, const void* w, uint32_t row,
                                           uint32_t rows, uint32_t heads, int sub) {
    const uint32_t rr = row < rows ? row : rows - 1;
    const uint32_t t = rr / heads, h = rr - t * heads;
    int64_t at;
    const bool ok = table_row(a, t, at);
    float y[8];
    turn<D, F16, float>(a, row_of(a, src, t, h), w, ok ? at : 0, sub, y);
    if (row >= rows) return;
    const uint4 o = pack8<F16>(y);
    reinterpret_cast<uint4*>(dst + static_cast<int64_t>(row) * D)[sub] = ok ? o : make_uint4(0, 0, 0, 0);
}

template <int D, bool F16>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
    constexpr int LPT = D / 8;
    const int sub = threadIdx.x & (LPT - 1);
    const uint32_t at = threadIdx.x / LPT;
    if (blockIdx.x < a.q_blocks) rotate_row<D, F16>(a, a.q, a.qo, a.qw, blockIdx.x * (256 / LPT) + at, a.tokens * a.hq, a.hq, sub);
    else rotate_row<D, F16>(a, a.k, a.ko, a.kw, (blockIdx.x - a.q_blocks) * (256 / LPT) + at, a.tokens * a.hk, a.hk, sub);
}

// The correctly rounded quotient x / s (s > 0 finite) from inv = RN(1 / s)
__device__ __forceinline__ double quot_rn(double x, double s, double inv) {
    const double q = x * inv;
    return __builtin_fma(__builtin_fma(-q, s, x), inv, q);
}

// A row of 4-bit codes: scale = fp16(fp32(max(amax, 1e-5) / 7)), code =
// RNE(x / scale).  Keys are rotated in 64 bits, so that the codes are those of
// the formula (a key next to a code's border by less than 32 bits' error would
// else fall on the wrong side).
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_rope_append_kernel(RopeArgs a) {
    constexpr int LPT = D / 8;
    const int sub = threadIdx.x & (LPT - 1);
    const uint32_t at = threadIdx.x / LPT;
    if (blockIdx.x < a.q_blocks) {
        rotate_row<D, F16>(a, a.q, a.qo, a.qw, blockIdx.x * (256 / LPT) + at, a.tokens * a.hq, a.hq, sub);
        return;
    }
    // (K and V rows of a token follow each other)
    const uint32_t row = (blockIdx.x - a.q_blocks) * (256 / LPT) + at, rows = a.tokens * a.hk * 2;
    const uint32_t rr = row < rows ? row : rows - 1;
    const uint32_t t = rr / (2 * a.hk), hh = rr - t * (2 * a.hk);
    const bool is_v = hh >= a.hk;
    const uint32_t h = is_v ? hh - a.hk : hh;
    const int64_t slot = a.pool.slots[t];
    int64_t tab;
    const bool ok = table_row(a, t, tab);
    _Float16 s16;
    uint32_t c[8];
    if (is_v) {
        float x[8], amax = 0.f;
        unpack8<F16>(reinterpret_cast<const uint4*>(row_of(a, a.v, t, h))[sub], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
        quant_row_codes<4>(x, fmaxf(lanes_max<LPT>(amax), 1e-5f), s16, c);
    } else {
        double x[8], amax = 0.0;
        turn<D, F16, double>(a, row_of(a, a.k, t, h), a.kw, ok ? tab : 0, sub, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmax(amax, fabs(x[i]));
        amax = fmax(lanes_max<LPT>(amax), 1e-5);
        s16 = static_cast<_Float16>(static_cast<float>(amax / 7.0));
        const double sf = static_cast<double>(s16), inv = 1.0 / sf;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double q = sf <= 65504.0 ? quot_rn(x[i], sf, inv) : x[i] / sf;
            c[i] = static_cast<uint32_t>(static_cast<int>(fmin(fmax(rint(q), -8.0), 7.0)));
        }
    }
    if (row >= rows || !ok || slot < 0 || slot >= a.pool.num_slots) return;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= (c[i] & 15u) << (4 * i);
    const int64_t page = slot >> a.pool.page_log2, off = slot & ((1 << a.pool.page_log2) - 1);
    int8_t* dst = (is_v ? a.pool.vp : a.pool.kp) + page * a.pool.ps_page + h * a.pool.ps_head + off * (D / 2);
    reinterpret_cast<uint32_t*>(dst)[sub] = word;
    if (sub == 0)
        static_cast<uint16_t*>(is_v ? a.pool.vs : a.pool.ks)[page * a.pool.ss_page + h * a.pool.ss_head + off] = __builtin_bit_cast(uint16_t, s16);
}

// ---------------------------------------------------------------------------
// 8-bit pages
// ---------------------------------------------------------------------------
// The exponent of a block's scale: the smallest e with max(amax, 1e-5) <= 127
// 2^e, so that x 2^-e and its rounding are exact and so are codes that are
// rounded again for a larger e.  Values past 127 2^MOST_E (and what is not
// finite) make the block's scale NaN.
constexpr int MOST_E = 40, BAD_E = 1 << 20, NO_E = -(1 << 20);
__device__ __forceinline__ int exponent(double amax) {
    if (!(amax <= 127.0 * 0x1p40)) return BAD_E;
    const uint64_t b = __builtin_bit_cast(uint64_t, fmax(amax, 1e-5));
    return static_cast<int>((b >> 52) & 2047) - 1022 - 7 + ((b & 0xfffffffffffffull) > 0xfc00000000000ull ? 1 : 0);
}
__device__ __forceinline__ int exponent(float amax) { return exponent(static_cast<double>(amax)); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// 16 tokens' new rows of one K or V head.  A run of tokens whose slots lie in one
// block is worked on by the workgroup that has its first token (31 rows at
// most): the block's scale is the largest that its new rows, and the rows before
// them, need; rows before the run's first live one (a token whose position is
// outside the table is not) stay, and are rounded again where the scale has
// grown.
template <int D, bool F16, bool ROPE>
__global__ __launch_bounds__(32 * (D / 8)) void paged8_append_kernel(RopeArgs a) {
    constexpr int LPT = D / 8, ROWS = 32;
    const int sub = threadIdx.x & (LPT - 1), r = threadIdx.x / LPT;
    if constexpr (ROPE) {
        if (blockIdx.x < a.q_blocks) {
            rotate_row<D, F16>(a, a.q, a.qo, a.qw, blockIdx.x * ROWS + r, a.tokens * a.hq, a.hq, sub);
            return;
        }
    }
    __shared__ int64_t slot_of[ROWS];
    __shared__ uint32_t starts, live;
    __shared__ int need[ROWS];
    const uint32_t i = blockIdx.x - a.q_blocks, win = i / (2 * a.hk), hh = i - win * (2 * a.hk);
    const bool is_v = hh >= a.hk;
    const uint32_t h = is_v ? hh - a.hk : hh, t0 = win * 16;
    if (threadIdx.x < 64) {              // tokens t0 - 1 .. t0 + 31
        const int64_t t = static_cast<int64_t>(t0) + threadIdx.x - 1;
        int64_t slot = -1;
        bool ok = true;
        if (threadIdx.x <= ROWS && t >= 0 && t < a.tokens) {
            slot = a.pool.slots[t];
            if (slot >= a.pool.num_slots || slot < 0) slot = -1;
            int64_t unused;
            if constexpr (ROPE) ok = table_row(a, static_cast<uint32_t>(t), unused);
        }
        const int64_t block = slot >> 4, before = __shfl_up(block, 1, 64);
        const uint64_t m = __builtin_amdgcn_ballot_w64(block != before), l = __builtin_amdgcn_ballot_w64(ok && slot >= 0);
        if (threadIdx.x == 0) { starts = static_cast<uint32_t>(m >> 1); live = static_cast<uint32_t>(l >> 1); }
        if (threadIdx.x >= 1 && threadIdx.x <= ROWS) slot_of[threadIdx.x - 1] = slot;
    }
    __syncthreads();
    const uint32_t upto = starts & (0xffffffffu >> (31 - r));
    const int run = upto ? 31 - __builtin_clz(upto) : -1;        // the run's first token, its live ones and the first of them
    const uint32_t more = run >= 0 && run < 31 ? starts & (0xfffffffeu << run) : 0;
    const uint32_t mine = run >= 0 ? live & (0xffffffffu << run) & (more ? (1u << __builtin_ctz(more)) - 1u : 0xffffffffu) : 0;
    const bool active = run < 16 && (mine >> r) & 1;
    const int first = mine ? __builtin_ctz(mine) : 0;
    const int64_t block = slot_of[r] >> 4;
    using T = std::conditional_t<ROPE, double, float>;
    T x[8];
    int e = NO_E;
    const uint32_t t = t0 + r;
    if (active) {
        if (is_v) unpack8<F16>(reinterpret_cast<const uint4*>(row_of(a, a.v, t, h))[sub], x);
        else if constexpr (!ROPE) unpack8<F16>(reinterpret_cast<const uint4*>(row_of(a, a.k, t, h))[sub], x);
        else {
            int64_t tab;
            table_row(a, t, tab);
            turn<D, F16, T>(a, row_of(a, a.k, t, h), a.kw, tab, sub, x);
        }
        T amax = 0;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const T y = x[j] < 0 ? -x[j] : x[j];
            bad |= !(y <= static_cast<T>(127.0 * 0x1p40));
            amax = y > amax ? y : amax;
        }
        e = lanes_max<LPT>(bad ? BAD_E : exponent(amax));
    }
    const int64_t page = block * BLOCK >> a.pool.page_log2;      // (an inactive row's address is not used)
    const int32_t off = static_cast<int32_t>(block * BLOCK & ((1 << a.pool.page_log2) - 1));
    int8_t* const rows = (is_v ? a.pool.vp : a.pool.kp) + page * a.pool.ps_page + h * a.pool.ps_head + off * D;
    float* const scale = static_cast<float*>(is_v ? a.pool.vs : a.pool.ks) + page * a.pool.ss_page + h * a.pool.ss_head + off / BLOCK;
    const int kept = active ? static_cast<int>(slot_of[first] & (BLOCK - 1)) : 0;
    const float old = kept ? *scale : 0.f;       // (read by all before the run's first row writes it)
    if (sub == 0) need[r] = e;
    __syncthreads();
    if (!active) return;
    for (uint32_t left = mine; left; left &= left - 1) e = max(e, need[__builtin_ctz(left)]);
    if (kept) {
        if (!(old >= 0.f && old <= pow2(MOST_E + 1))) e = BAD_E;
        else if (old > 0.f) {            // the smallest power of two from it on
            const uint32_t b = __float_as_uint(old);
            e = max(e, static_cast<int>(b >> 23) - 127 + (b & 0x7fffffu ? 1 : 0));
        }
    }
    const bool bad = e > MOST_E + 1;
    const float now = bad ? __builtin_nanf("") : pow2(e), inv = bad ? 0.f : pow2(-e);
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (ROPE) c[j] = static_cast<uint32_t>(static_cast<int>(rint(x[j] * static_cast<double>(inv)))) & 255u;
        else c[j] = static_cast<uint32_t>(static_cast<int>(rintf(x[j] * inv))) & 255u;
    }
    const uint2 word = make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
    const int row = static_cast<int>(slot_of[r] & (BLOCK - 1));
    reinterpret_cast<uint2*>(rows + row * D)[sub] = word;
    if (r != first) return;
    if (kept && now != old) {
        const float by = old * inv;
        for (int j = 0; j < kept; ++j) {
            uint2* const p = reinterpret_cast<uint2*>(rows + j * D) + sub;
            const uint2 w = *p;
            const uint32_t in[2] = {w.x, w.y};
            uint32_t out[2] = {0, 0};
#pragma unroll
            for (int i8 = 0; i8 < 8; ++i8) {
                const int code = static_cast<int8_t>(in[i8 >> 2] >> (8 * (i8 & 3)));
                const int again = static_cast<int>(rintf(static_cast<float>(code) * by));
                out[i8 >> 2] |= (static_cast<uint32_t>(again) & 255u) << (8 * (i8 & 3));
            }
            *p = make_uint2(out[0], out[1]);
        }
    }
    if (sub == 0) *scale = now;
}

// Rows of the cache by slot as bf16 or fp16 values, code * scale rounded once
// (exact for bf16); slots outside the pool give zero rows.
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
    reinterpret_cast<uint4*>((is_v ? ov : ok) + static_cast<int64_t>(row) * D)[sub] = pack8<F16>(y);
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
    const int64_t most = MOST_THREADS / (p->head_dim / 8), heads = std::max(p->q_heads + 4 * p->k_heads, 1);
    if (p->n > most || p->batch > most || (p->n && p->batch > most / p->n) || p->batch * p->n > (most / heads) - 32)
        return fail(HYQ_ENOTSUP, w + "more than " + std::to_string(most) + " rows");
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

template <bool ROPE>
int launch_append8(RopeArgs a, int head_dim, bool fp16, hipStream_t st) {
    a.q_blocks = ROPE ? blocks_of(static_cast<uint64_t>(a.tokens) * a.hq, 32) : 0;
    const dim3 grid(a.q_blocks + blocks_of(a.tokens, 16) * a.hk * 2);
    if (head_dim == 128) {
        if (fp16) paged8_append_kernel<128, true, ROPE><<<grid, dim3(512), 0, st>>>(a);
        else paged8_append_kernel<128, false, ROPE><<<grid, dim3(512), 0, st>>>(a);
    } else {
        if (fp16) paged8_append_kernel<64, true, ROPE><<<grid, dim3(256), 0, st>>>(a);
        else paged8_append_kernel<64, false, ROPE><<<grid, dim3(256), 0, st>>>(a);
    }
    return check_launch("hyq_paged8_append");
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
    RopeArgs a = args_of(*p);
    const unsigned per = 256 / (p->head_dim / 8);
    a.q_blocks = blocks_of(static_cast<uint64_t>(a.tokens) * a.hq, per);
    const unsigned grid = a.q_blocks + blocks_of(static_cast<uint64_t>(a.tokens) * a.hk, per);
    if (a.tokens == 0 || grid == 0) return HYQ_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p->head_dim == 128) {
        if (p->dtype_fp16) qk_norm_rope_kernel<128, true><<<dim3(grid), dim3(256), 0, st>>>(a);
        else qk_norm_rope_kernel<128, false><<<dim3(grid), dim3(256), 0, st>>>(a);
    } else {
        if (p->dtype_fp16) qk_norm_rope_kernel<64, true><<<dim3(grid), dim3(256), 0, st>>>(a);
        else qk_norm_rope_kernel<64, false><<<dim3(grid), dim3(256), 0, st>>>(a);
    }
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
    if (pool->bits == 8) return launch_append8<true>(a, p->head_dim, p->dtype_fp16, st);
    const unsigned per = 256 / (p->head_dim / 8);
    a.q_blocks = blocks_of(static_cast<uint64_t>(a.tokens) * a.hq, per);
    const dim3 grid(a.q_blocks + blocks_of(static_cast<uint64_t>(a.tokens) * a.hk * 2, per));
    if (p->head_dim == 128) {
        if (p->dtype_fp16) paged_rope_append_kernel<128, true><<<grid, dim3(256), 0, st>>>(a);
        else paged_rope_append_kernel<128, false><<<grid, dim3(256), 0, st>>>(a);
    } else {
        if (p->dtype_fp16) paged_rope_append_kernel<64, true><<<grid, dim3(256), 0, st>>>(a);
        else paged_rope_append_kernel<64, false><<<grid, dim3(256), 0, st>>>(a);
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
    if (num_tokens > most / (4 * kv_heads) - 32) return fail(HYQ_ENOTSUP, w + "more than " + std::to_string(most) + " rows");
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
    return launch_append8<false>(a, head_dim, is_fp16, static_cast<hipStream_t>(stream));
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
