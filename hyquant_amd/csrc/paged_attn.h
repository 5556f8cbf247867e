// What the paged caches' attention kernels share: the schedule of a ragged batch,
// a tile's rows and their pieces, the join of the pieces, and the host side.
#pragma once

#include "hyq_common.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <string>

namespace hyq {

// Calls with counters are numbered in the order of their launches, whichever
// cache they read: they may share a stream's counters.
struct CallOrder {
    std::mutex mutex;
    uint64_t calls = 0;
};
CallOrder& call_order();

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int MIN_PAGE = 16, MAX_PAGE = 256;

bool ok_page(int page) { return page >= MIN_PAGE && page <= MAX_PAGE && (page & (page - 1)) == 0; }
int log2i(int x) {
    int l = 0;
    while ((1 << l) < x) ++l;
    return l;
}

// the last i in [0, n] with a[i] <= x (a[0] <= x, a ascending)
template <typename T>
__device__ __forceinline__ int last_at_most(const T* a, int n, T x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// inclusive sums over the wavefront by DPP row shifts and broadcasts
__device__ __forceinline__ int scan_dpp(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);    // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);    // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);    // row_bcast:31 into rows 2 and 3
    return v;
}

template <typename T>
__device__ __forceinline__ T wave_incl_scan(T v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float xmax16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xmax32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float col_max(float v) { return xmax32(xmax16(v)); }
__device__ __forceinline__ float col_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------------------------------
// attention: the schedule
// ---------------------------------------------------------------------------
// Query rows of a request are its new tokens times the G query heads of a KV
// head, row = token * G + head, cut into tiles of TILE rows; a tile's keys may
// be cut into pieces, whose partial results a join launch adds up.  The
// schedule is the same for every KV head.  It is made on the device from the
// lengths, so that nothing is read back and a captured graph follows the
// lengths it is replayed with: up to 256 requests every wavefront finds its own
// item (a lane looks at one request, or at four neighbours where there are more
// than 64; one round of loads, a few wavefront scans), more are laid out by a
// launch before.
// Requests of at most 16 rows (decode steps) and larger ones (chunks) have a
// kernel and a schedule each: a tile of 16 rows is bound by the cache's bytes,
// one of CHUNK rows by the products.
constexpr int PLAN_T = 1024;
constexpr int LANE_R = 4;                // requests of a lane, at most
constexpr int INLINE_R = 64 * LANE_R;    // requests of a schedule without a launch of its own
constexpr int JOIN_T = 1024;             // threads of a join's workgroup
constexpr int CHUNK_WAVES = 8;
constexpr int CHUNK = 32 * CHUNK_WAVES;  // rows of a chunk tile
struct Narrow {
    static constexpr int TILE = 16, GROUP = 32;   // query rows per tile, keys per step
    static constexpr int MIN_UNITS = 12;          // steps per piece, at least: each wavefront's ring of loads full once
    static constexpr float UNCUT = 1.5f;          // pieces that a tile has to be longer than, to be cut
    static constexpr int join_rows(int lane_groups) { return lane_groups / 4; }   // rows of a join's workgroup
    static constexpr int slots(int head_dim) { return head_dim == 64 ? 1024 : 768; }   // resident workgroups
    static __host__ __device__ bool few(float target, float tiles) { return tiles <= 0.4f * target; }
    static __host__ __device__ float wanted(float target, float tiles) {
        return few(target, tiles) ? target - 0.5f * tiles : 1.333f * target;
    }
    static __host__ __device__ float uncut(float target, float tiles) { return few(target, tiles) ? UNCUT : 2.1f; }
    static int64_t most(int64_t target, int64_t tiles) { return few(target, tiles) ? target : target + target / 3 + 1; }
};
struct Wide {
    static constexpr int TILE = CHUNK, GROUP = 64;
    static constexpr int MIN_UNITS = 4;
    static constexpr float UNCUT = 1.15f;
    static constexpr int join_rows(int lane_groups) { return lane_groups; }
    static constexpr int slots(int) { return 256; }
    static __host__ __device__ float wanted(float target, float tiles) { return fmaxf(target - 0.5f * tiles, 0.5f * target); }
    static __host__ __device__ float uncut(float, float) { return UNCUT; }
    static int64_t most(int64_t target, int64_t) { return target; }
};

struct Item {
    int32_t req, q0, qlen, len;          // request, its first token, its new tokens, its keys
    int32_t row0;                        // first row of the tile within the request
    int32_t key0, key1;                  // keys of this piece
    int32_t part;                        // partial slot, -1: the tile is whole
    int32_t join, part0, pieces;         // of a cut tile: its join, its first partial slot, its pieces
    int32_t pad;
};
struct Join {
    int32_t q0, row0, rows, part, pieces, pad[3];
};
struct Counts {
    int32_t items, joins, pad[2];
};

struct PlanArgs {
    const int32_t* lens;
    const int32_t* cu;
    int32_t R, T, G, window, capacity;   // capacity: keys that a block table row can name
    int32_t target;                      // pieces per KV head wanted
    int32_t max_items, max_parts, max_joins;
    Counts* counts;
    Item* items;
    Join* joins;
};

struct Req {
    int32_t q0, qlen, len, tiles, units; // units: the longest tile's GROUP-key steps
};

// first key that a row at position pos sees
__device__ __forceinline__ int first_key(int pos, int window) { return window > 0 ? max(0, pos - window + 1) : 0; }

template <typename K>
__device__ __forceinline__ Req request(const PlanArgs& a, int r) {
    Req q{};
    if (r >= a.R) return q;
    q.q0 = r;
    q.qlen = 1;
    if (a.cu) {
        q.q0 = min(max(a.cu[r], 0), a.T);
        q.qlen = min(max(a.cu[r + 1], q.q0), a.T) - q.q0;
    }
    q.len = min(max(a.lens[r], 0), a.capacity);
    const int rows = q.qlen * a.G;
    q.tiles = (rows <= Narrow::TILE) == (K::TILE == Narrow::TILE) ? (rows + K::TILE - 1) / K::TILE : 0;
    // the rows of a tile see at most window + TILE keys between them
    const int keys = a.window > 0 && a.window < q.len - K::TILE ? a.window + K::TILE : q.len;
    q.units = keys / K::GROUP + 2;       // from a GROUP boundary to a GROUP boundary
    return q;
}

// GROUP steps per piece.  A slot is a resident workgroup (`target` of them per KV
// head).  Where tiles are few, the pieces are to fill the slots exactly once:
// rounding up makes half a piece more per tile, so that many slots are kept
// back.  Where 16-row tiles are many, that would make the pieces long and
// unequal: a third more pieces than slots are cut, and the last ones fill up.
// A tile that is hardly longer than a piece is not cut, it would cost the
// partial results for nothing.  Measured on requests of 128 channels, 8 KV heads
// (decode steps with a weight in one bf16 number; in two they take 3 to 6% more):
//   16 requests of 8K keys    exactly one round 33 us, 1024 pieces and more 39
//   24 requests of 16K        77, 85
//   64 requests of 1K to 32K  one round 163, a third more 123, twice as many 120
//   48 requests of 0.7 to 32K one round 92, a third more 87
//   64 requests of 1K         cut in two 31, whole 24
//   one request of 8K         12 steps at least 12.6, 8 steps 14.6, 16 steps 13.8
//   4 chunks of 100 to 700 tokens at 2K to 9K: wide pieces for one round 206,
//                             for three quarters of one 253
// (The float sum's rounding is far below 2^-14.)
template <typename K>
__device__ __forceinline__ int units_per_piece(const PlanArgs& a, float work, float tiles, float longest) {
    const float target = static_cast<float>(a.target);
    const float per = fmaxf(ceilf(work * (1.0f + 0x1p-14f) / K::wanted(target, tiles)), static_cast<float>(K::MIN_UNITS));
    if (longest <= per * K::uncut(target, tiles)) return 1 << 30;
    return static_cast<int>(fminf(per, 0x1p30f));
}
__device__ __forceinline__ int pieces_of(const Req& x, int per) {
    return static_cast<int>((static_cast<uint32_t>(x.units) + static_cast<uint32_t>(per) - 1u) / static_cast<uint32_t>(per));
}

// Piece `piece` of pc of tile `tile` of a request
template <typename K>
__device__ __forceinline__ Item make_item(const PlanArgs& a, const Req& x, int r, int tile, int piece, int pc,
                                          int part0, int join) {
    const int row0 = tile * K::TILE, row1 = min(row0 + K::TILE, x.qlen * a.G);
    const int p0 = x.len - x.qlen + row0 / a.G, p1 = x.len - x.qlen + (row1 - 1) / a.G;   // first and last position
    const int lo = first_key(p0, a.window) / K::GROUP, hi = (max(p1, -1) + K::GROUP) / K::GROUP;   // GROUP steps
    const int steps = max(hi - lo, 0), each = static_cast<int>((static_cast<uint32_t>(steps) + pc - 1u) / pc);
    Item it{r, x.q0, x.qlen, x.len, row0, 0, 0, part0 >= 0 ? part0 + piece : -1, join, part0, pc, 0};
    it.key0 = (lo + min(steps, piece * each)) * K::GROUP;
    it.key1 = min(p1 + 1, (lo + min(steps, (piece + 1) * each)) * K::GROUP);
    return it;
}
template <typename K>
__device__ __forceinline__ Join make_join(const PlanArgs& a, const Req& x, int tile, int pc, int part) {
    return Join{x.q0, tile * K::TILE, min(K::TILE, x.qlen * a.G - tile * K::TILE), part, pc, {0, 0, 0}};
}

__device__ __forceinline__ float wave_top(float v) {
    v = col_max(max16_dpp(v));
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = col_sum(sum16_dpp(v));
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

// The schedule of up to INLINE_R requests in one wavefront's registers.  32 bits
// are enough whatever the lengths: 256 requests of at most 2^22 tiles each and
// the target's pieces on top.
struct RegPlan {
    Req x[LANE_R];                       // of the lane's requests
    int pc[LANE_R];
    int items, parts, joins;             // before them
    int r0, n;                           // the lane's first request and how many a lane has (the same in every lane)
};
template <typename K>
__device__ __forceinline__ RegPlan reg_plan(const PlanArgs& a, int lane) {
    RegPlan p;
    p.n = a.R <= 64 ? 1 : LANE_R;
    p.r0 = lane * p.n;
    float work = 0.f, tiles = 0.f, longest = 0.f;
#pragma unroll
    for (int j = 0; j < LANE_R; ++j) {
        p.x[j] = Req{0, 0, 0, 0, 0};
        if (j < p.n) p.x[j] = request<K>(a, p.r0 + j);
    }
#pragma unroll
    for (int j = 0; j < LANE_R; ++j) {
        tiles += static_cast<float>(p.x[j].tiles);
        work += static_cast<float>(p.x[j].tiles) * static_cast<float>(p.x[j].units);
        if (p.x[j].tiles) longest = fmaxf(longest, static_cast<float>(p.x[j].units));
    }
    const int per = units_per_piece<K>(a, wave_sum(work), wave_sum(tiles), wave_top(longest));
    int items = 0, parts = 0, joins = 0;
#pragma unroll
    for (int j = 0; j < LANE_R; ++j) {
        p.pc[j] = 1;
        if (j < p.n) {
            p.pc[j] = pieces_of(p.x[j], per);
            const int n = p.x[j].tiles * p.pc[j], split = p.pc[j] > 1 ? 1 : 0;
            items += n;
            parts += split * n;
            joins += split * p.x[j].tiles;
        }
    }
    p.items = scan_dpp(items) - items;
    p.parts = scan_dpp(parts) - parts;
    p.joins = scan_dpp(joins) - joins;
    return p;
}

// This workgroup's item; false: it has none.  With `head` 0 it also leaves what
// the join launch reads: a split tile's first piece its join, workgroup 0 how
// many there are, of requests that fit the limits whole (offsets that do not
// ascend may name more tiles than the grid has).
template <typename K>
__device__ __forceinline__ bool find_item(const PlanArgs& a, int i, int head, int lane, Item& it) {
    if (a.R > INLINE_R) {
        if (i >= a.counts->items) return false;
        it = a.items[i];
        return true;
    }
    const RegPlan p = reg_plan<K>(a, lane);
    // the lane and request that entry i belongs to
    Req x{};
    int r = 0, pc = 1, local = 0, part = 0, join = 0;
    bool any = false;
    int whole = 0;
    int at = p.items, parts = p.parts, joins = p.joins;
#pragma unroll
    for (int j = 0; j < LANE_R; ++j) {
        if (j < p.n) {
            const int n = p.x[j].tiles * p.pc[j];
            if (at <= i && i < at + n) {
                x = p.x[j];
                r = p.r0 + j;
                pc = p.pc[j];
                local = i - at;
                part = parts;
                join = joins;
                any = true;
            }
            at += n;
            parts += p.pc[j] > 1 ? n : 0;
            joins += p.pc[j] > 1 ? p.x[j].tiles : 0;
            if (at <= a.max_items && parts <= a.max_parts) whole = min(joins, a.max_joins);
        }
    }
    if (i == 0 && head == 0) {
        const float top = wave_top(static_cast<float>(whole));         // (at most 1024 joins)
        if (threadIdx.x == 0) a.counts->joins = static_cast<int>(top);
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(any);
    if (!m) return false;
    const int k = __builtin_ctzll(m);
    auto get = [&](int v) { return __builtin_amdgcn_readlane(v, k); };
    x = Req{get(x.q0), get(x.qlen), get(x.len), get(x.tiles), get(x.units)};
    pc = get(pc);
    local = get(local);
    // (a causal request's last tiles have the most keys: they go first)
    const int nth = local / pc, piece = local - nth * pc;
    part = get(part) + nth * pc;
    join = get(join) + nth;
    const bool split = pc > 1 && part + pc <= a.max_parts && join < a.max_joins;
    it = make_item<K>(a, x, get(r), x.tiles - 1 - nth, piece, pc, split ? part : -1, join);
    if (split && piece == 0 && head == 0 && threadIdx.x == 0) a.joins[join] = make_join<K>(a, x, x.tiles - 1 - nth, pc, part);
    return true;
}

template <typename K>
__device__ __forceinline__ void plan(const PlanArgs& a) {
    // items, partial slots and joins before each request of a round (64 bits:
    // lengths that make no sense may add up to anything)
    __shared__ int64_t start[3][PLAN_T];
    __shared__ int64_t wsum[3][PLAN_T / 64];
    __shared__ int whole;                // joins of requests that fit the limits whole
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    __shared__ float fsum[3][PLAN_T / 64];
    float work = 0.f, tiles = 0.f, longest = 0.f;
    for (int r = tid; r < a.R; r += PLAN_T) {
        const Req q = request<K>(a, r);
        tiles += static_cast<float>(q.tiles);
        work += static_cast<float>(q.tiles) * static_cast<float>(q.units);
        if (q.tiles) longest = fmaxf(longest, static_cast<float>(q.units));
    }
    work = wave_sum(work);
    tiles = wave_sum(tiles);
    longest = wave_top(longest);
    if (lane == 0) { fsum[0][w] = work; fsum[1][w] = longest; fsum[2][w] = tiles; }
    if (tid == 0) whole = 0;
    __syncthreads();
    work = tiles = longest = 0.f;
    for (int i = 0; i < PLAN_T / 64; ++i) { work += fsum[0][i]; longest = fmaxf(longest, fsum[1][i]); tiles += fsum[2][i]; }
    __syncthreads();
    const int per = units_per_piece<K>(a, work, tiles, longest);
    int64_t base[3] = {0, 0, 0};
    for (int r0 = 0; r0 < a.R; r0 += PLAN_T) {
        const Req q = request<K>(a, r0 + tid);
        const int64_t pieces = pieces_of(q, per);
        const int64_t n[3] = {q.tiles * pieces, pieces > 1 ? q.tiles * pieces : 0, pieces > 1 ? q.tiles : 0};
        int64_t incl[3], total[3] = {0, 0, 0};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            incl[k] = wave_incl_scan(n[k], lane);
            if (lane == 63) wsum[k][w] = incl[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            int64_t before = 0;
            for (int i = 0; i < PLAN_T / 64; ++i) {
                if (i < w) before += wsum[k][i];
                total[k] += wsum[k][i];
            }
            start[k][tid] = before + incl[k] - n[k];
            incl[k] += base[k] + before;
        }
        if (n[2] && incl[0] <= a.max_items && incl[1] <= a.max_parts)
            atomicMax(&whole, static_cast<int>(min(incl[2], static_cast<int64_t>(a.max_joins))));
        __syncthreads();
        const int nr = min(PLAN_T, a.R - r0);
        for (int64_t i = tid; i < total[0] && base[0] + i < a.max_items; i += PLAN_T) {
            const int k = last_at_most(start[0], nr - 1, i);
            const Req x = request<K>(a, r0 + k);
            const int pc = pieces_of(x, per), local = static_cast<int>(i - start[0][k]), nth = local / pc, piece = local - nth * pc;
            const int tile = x.tiles - 1 - nth;
            const int64_t part = base[1] + start[1][k] + local - piece, j = base[2] + start[2][k] + nth;
            const bool split = pc > 1 && part + pc <= a.max_parts && j < a.max_joins;
            a.items[base[0] + i] = make_item<K>(a, x, r0 + k, tile, piece, pc, split ? static_cast<int>(part) : -1, static_cast<int>(j));
            if (split && piece == 0) a.joins[j] = make_join<K>(a, x, tile, pc, static_cast<int>(part));
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) base[k] += total[k];
        __syncthreads();
    }
    if (tid == 0) *a.counts = Counts{static_cast<int32_t>(min(base[0], static_cast<int64_t>(a.max_items))), whole, {0, 0}};
}
// block 0: the schedule of the short requests, block 1: the chunks'
__global__ __launch_bounds__(PLAN_T) void paged_plan_kernel(PlanArgs narrow, PlanArgs wide) {
    if (blockIdx.x == 0) plan<Narrow>(narrow);
    else plan<Wide>(wide);
}

struct AttnArgs {
    const uint16_t* q;
    int64_t q_t, q_h;
    uint16_t* out;
    int64_t o_t, o_h;
    float* lse;
    int64_t l_t;
    const int8_t *kp, *vp;
    int64_t ps_page, ps_head;
    const void *ks, *vs;
    int64_t ss_page, ss_head;
    const int32_t* table;
    int64_t bt_stride;
    PlanArgs plan;
    float* part;                         // [slot][key head][TILE][D] sums; ml: [slot][key head][TILE][2] (m, l)
    float* ml;
    uint64_t* counters;                  // arrivals per join and KV head (the last workgroup joins), or null: a launch joins
    uint64_t call;                       // this call's number << CALL_SHIFT
    int32_t G, heads, page_log2, num_pages, window, zero_tail;
    float scale;                         // sm_scale * log2(e)
};

constexpr float M_INIT = -3.0e38f;       // below any score
constexpr float SLACK = 8.0f;            // the running maximum moves when a score passes it by this (log2 units)
constexpr int WAVES = 4;                 // of the 16-row kernel
constexpr float LN2 = 0.69314718055994531f;

// 16-bit words of a row as floats (exact)
template <bool F16>
__device__ __forceinline__ float half_at(uint32_t w, int hi) {
    if constexpr (F16) return f16_bits_to_f32(static_cast<uint16_t>(hi ? w >> 16 : w));
    else return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
}

// The power of two that brings a row's largest magnitude (or that of many rows)
// to [2^14, 2^15), so that fp16 holds the queries exactly down to 2^-38 of it;
// returned as the exponent to subtract, in [-114, 113].
__device__ __forceinline__ int q_exponent(float amax) {
    const int e = static_cast<int>((__float_as_uint(amax) >> 23) & 255u) - 127;
    return max(e, -100) - 14;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// out (and lse) of a row from its sums: a row without keys is zero, NaN stays NaN
template <bool F16>
__device__ __forceinline__ void store_row(const AttnArgs& a, int q0, int rr, int head, int ch, float m, float l, f32x4 o) {
    const int tk = rr / a.G;
    const int64_t h = static_cast<int64_t>(head) * a.G + rr - tk * a.G, t = static_cast<int64_t>(q0) + tk;
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
    o *= inv;
    u32x2 ow;
    if constexpr (F16) {
        ow[0] = f32_to_f16_bits(o[0]) | (static_cast<uint32_t>(f32_to_f16_bits(o[1])) << 16);
        ow[1] = f32_to_f16_bits(o[2]) | (static_cast<uint32_t>(f32_to_f16_bits(o[3])) << 16);
    } else {
        ow[0] = pack_bf16x2(o[0], o[1]);
        ow[1] = pack_bf16x2(o[2], o[3]);
    }
    *reinterpret_cast<u32x2*>(a.out + t * a.o_t + h * a.o_h + ch) = ow;
    if (a.lse && ch == 0) a.lse[t * a.l_t + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// ---- adding up pieces ----
// The pieces of a row of a 16-row tile are eight interleaved streams, each added
// in order, and the streams a binary tree: the same sums whichever kernel adds
// them and however many threads share a row.  A 256-row tile's few pieces are
// added in order.
struct Sum {
    float m, l;
    f32x4 o;
};
__device__ __forceinline__ Sum add(const Sum& x, const Sum& y) {
    const float m = fmaxf(x.m, y.m), fx = fast_exp2(x.m - m), fy = fast_exp2(y.m - m);
    return Sum{m, x.l * fx + y.l * fy, x.o * fx + y.o * fy};
}

typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr int NT = 2;                    // cache policy bit: non-temporal (codes are read once)
__device__ __forceinline__ Rsrc make_rsrc(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}

constexpr int COUNTER_PAD = 16;          // a counter has a 128-byte line: arrivals at one line queue up
constexpr int CALL_SHIFT = 16;           // a counter is the call's number and its arrivals (at most 1366 pieces)
constexpr int SC1 = 16;                  // cache policy bit: device scope

// Streams s0 .. s0 + VS - 1 of a row's pieces at this lane's 4 channels: `o` and
// `ml` describe the pieces' sums and (m, l), the lane's own at byte offsets
// oat and mat, the next piece's ostep and mstep further (past the last one the
// loads are out of range: zeros, no access).  `DEEP` pieces in flight.
template <int VS, int DEEP, int POLICY, int STREAMS = 8>
__device__ __forceinline__ Sum add_streams(Rsrc o, Rsrc ml, uint32_t oat, uint32_t mat, uint32_t ostep, uint32_t mstep,
                                           int pieces, int s0) {
    constexpr int RD = DEEP / VS;
    Sum s[VS];
#pragma unroll
    for (int v = 0; v < VS; ++v) s[v] = Sum{M_INIT, 0.f, {0.f, 0.f, 0.f, 0.f}};
    for (int i0 = s0; i0 < pieces; i0 += STREAMS * RD) {
        Sum x[RD][VS];
#pragma unroll
        for (int r = 0; r < RD; ++r)
#pragma unroll
            for (int v = 0; v < VS; ++v) {
                const uint32_t p = static_cast<uint32_t>(i0 + STREAMS * r + v);
                const u32x2 t = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(ml, mat + p * mstep, 0, POLICY));
                x[r][v] = Sum{__uint_as_float(t[0]), __uint_as_float(t[1]),
                              __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(o, oat + p * ostep, 0, POLICY))};
            }
#pragma unroll
        for (int r = 0; r < RD; ++r)
#pragma unroll
            for (int v = 0; v < VS; ++v)
                if (i0 + STREAMS * r + v < pieces) s[v] = add(s[v], x[r][v]);
    }
#pragma unroll
    for (int d = 1; d < VS; d *= 2)
#pragma unroll
        for (int v = 0; v < VS; v += 2 * d) s[v] = add(s[v], s[v + d]);
    return s[0];
}

// The wavefronts' results of a 16-row tile, joined through LDS: red [wavefront][row]
// [channel], their maxima and sums.  Where the tile is cut and there are counters,
// the tile's last workgroup adds up its pieces.
template <int D, bool F16>
__device__ __forceinline__ void finish_tile(const AttnArgs& a, const Item& it, int head, int nrows,
                                            float (&red)[WAVES][Narrow::TILE][D + 4], float (&redm)[WAVES][Narrow::TILE],
                                            float (&redl)[WAVES][Narrow::TILE]) {
    constexpr int TILE = Narrow::TILE;
    const int tid = threadIdx.x;
    __syncthreads();
    for (int e = tid; e < nrows * (D / 4); e += 64 * WAVES) {
        const int rw = e / (D / 4), ch = 4 * (e - rw * (D / 4));
        float m = redm[0][rw];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) m = fmaxf(m, redm[i][rw]);
        float l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const float f = fast_exp2(redm[i][rw] - m);
            l += f * redl[i][rw];
            o += f * *reinterpret_cast<const f32x4*>(&red[i][rw][ch]);
        }
        if (it.part >= 0) {              // (device scope: another XCD's workgroup may read them in this launch)
            const int64_t slot = static_cast<int64_t>(it.part) * a.heads + head;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), make_rsrc(a.part + slot * TILE * D, TILE * D * 4),
                                                   (rw * D + ch) * 4, 0, SC1);
            if (ch == 0) {
                __hip_atomic_store(a.ml + (slot * TILE + rw) * 2, m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(a.ml + (slot * TILE + rw) * 2 + 1, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        } else {
            store_row<F16>(a, it.q0, it.row0 + rw, head, ch, m, l, o);
        }
    }
    if (!a.counters || it.part < 0) return;

    // ---- the tile's last workgroup adds up its pieces ----
    // every store of this workgroup is acknowledged before its arrival is counted
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    __shared__ int last;
    // (arrivals that an earlier call left behind, because its lengths were changed
    // while it ran, are below this call's number: the maximum takes them away)
    uint64_t* const counter = a.counters + (static_cast<int64_t>(it.join) * a.heads + head) * COUNTER_PAD;
    if (tid == 0) {
        (void)__hip_atomic_fetch_max(counter, a.call, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(counter, uint64_t{1}, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.call + it.pieces - 1;
        if (last) __hip_atomic_store(counter, uint64_t{0}, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    constexpr int LG = 64 * WAVES / (D / 4);       // lane groups of a row
    const int g = tid / (D / 4), ch = 4 * (tid - g * (D / 4));
    const uint32_t pieces = it.pieces, ostep = a.heads * (TILE * D * 4), mstep = a.heads * (TILE * 2 * 4);
    const int64_t slot0 = static_cast<int64_t>(it.part0) * a.heads + head;
    const Rsrc ro = make_rsrc(a.part + slot0 * TILE * D, (pieces - 1) * ostep + TILE * D * 4);
    const Rsrc rm = make_rsrc(a.ml + slot0 * TILE * 2, (pieces - 1) * mstep + TILE * 2 * 4);
    if (nrows <= LG / 2) {               // two lane groups share a row
        const int rw = g >> 1;
        Sum s{M_INIT, 0.f, {0.f, 0.f, 0.f, 0.f}};
        if (rw < nrows) s = add_streams<4, 8, SC1>(ro, rm, (rw * D + ch) * 4, rw * 8, ostep, mstep, it.pieces, 4 * (g & 1));
        float* const other = &red[0][0][0] + rw * (D + 4) + ch;
        if (g & 1) {
            *reinterpret_cast<f32x4*>(other) = s.o;
            if (ch == 0) { redm[0][rw] = s.m; redl[0][rw] = s.l; }
        }
        __syncthreads();
        if (!(g & 1) && rw < nrows) {
            s = add(s, Sum{redm[0][rw], redl[0][rw], *reinterpret_cast<const f32x4*>(other)});
            store_row<F16>(a, it.q0, it.row0 + rw, head, ch, s.m, s.l, s.o);
        }
    } else {
        for (int rw = g; rw < nrows; rw += LG) {
            const Sum s = add_streams<8, 8, SC1>(ro, rm, (rw * D + ch) * 4, rw * 8, ostep, mstep, it.pieces, 0);
            store_row<F16>(a, it.q0, it.row0 + rw, head, ch, s.m, s.l, s.o);
        }
    }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
constexpr float P_SHIFT = 6.0f;          // P' is at most 2^(P_SHIFT + SLACK_W + 1)
constexpr float SLACK_W = 6.0f;
constexpr int BLK = 64;                  // keys per block
constexpr int BUFS = 3;                  // blocks in LDS

// Bytes from a key's row of D fp16 channels to the next's.  16 lanes of a K
// operand read (neighbouring rows, one 16-byte chunk) and 32 of a transposing V
// read (4 rows, 64 bytes) fall on all 64 banks once by the padding, so a lane's
// operands are one address and constants.
template <int D> constexpr int KROW = 2 * D + 16;
template <int D> constexpr int VROW = 2 * D + 64;

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
    const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}


// Adds up the pieces of the split tiles, of both kinds in one launch (`blocks`
// of the grid take the short requests').  A workgroup takes some rows of a tile
// and KV head after the other; a row is 4 channels a lane of D/4, and 4 or 8 lane
// groups share the pieces of a short request's row and meet in LDS.  Four pieces are in flight per lane (with eight one
// workgroup a CU is resident instead of two: 15 us instead of 7 beside chunks).  By zero_tail
// it also clears the rows behind the last request.
template <int D>
struct JoinLds {
    static constexpr int LG = JOIN_T / (D / 4);    // lane groups
    float so[LG][D];
    float sm[LG], sl[LG];
};

template <typename K, int D, bool F16>
__device__ __forceinline__ void join_tiles(const AttnArgs& a, JoinLds<D>& L, int block, int blocks) {
    constexpr int LG = JoinLds<D>::LG;
    constexpr int ROWS = K::join_rows(LG), PARTS = K::TILE / ROWS;     // of a tile
    constexpr bool NARROW = K::TILE == Narrow::TILE;
    const int tid = threadIdx.x;
    const int g = tid / (D / 4), ch = 4 * (tid - g * (D / 4));
    if (a.plan.max_joins == 0) return;   // (nothing can be cut, and where the kind has no tiles nobody wrote the counts)
    const int64_t total = static_cast<int64_t>(a.plan.counts->joins) * a.heads * PARTS;
    for (int64_t i = block; i < total; i += blocks) {
        const uint32_t rest = static_cast<uint32_t>(i) / a.heads;
        const int head = static_cast<uint32_t>(i) - rest * a.heads;
        const Join jn = a.plan.joins[rest / PARTS];
        const int first = rest % PARTS * ROWS, rows = min(ROWS, jn.rows - first);
        const int share = NARROW ? rows <= LG / 8 ? 8 : 4 : 1;         // lane groups of a row
        const int sub = g % share, rw = g / share;
        const uint32_t ostep = a.heads * (K::TILE * D * 4), mstep = a.heads * (K::TILE * 2 * 4);
        const int64_t slot0 = static_cast<int64_t>(jn.part) * a.heads + head;
        Sum s{M_INIT, 0.f, {0.f, 0.f, 0.f, 0.f}};
        if (rw < rows) {
            const Rsrc ro = make_rsrc(a.part + slot0 * K::TILE * D, (jn.pieces - 1) * ostep + K::TILE * D * 4);
            const Rsrc rm = make_rsrc(a.ml + slot0 * K::TILE * 2, (jn.pieces - 1) * mstep + K::TILE * 2 * 4);
            const uint32_t oat = ((first + rw) * D + ch) * 4, mat = (first + rw) * 8;
            if (!NARROW) s = add_streams<1, 4, 0, 1>(ro, rm, oat, mat, ostep, mstep, jn.pieces, 0);
            else if (share == 8) s = add_streams<1, 4, 0>(ro, rm, oat, mat, ostep, mstep, jn.pieces, sub);
            else s = add_streams<2, 4, 0>(ro, rm, oat, mat, ostep, mstep, jn.pieces, 2 * sub);
        }
        for (int d = 1; d < share; d *= 2) {
            if (sub & d) {
                *reinterpret_cast<f32x4*>(&L.so[g][ch]) = s.o;
                if (ch == 0) { L.sm[g] = s.m; L.sl[g] = s.l; }
            }
            __syncthreads();
            if (!(sub & (2 * d - 1))) s = add(s, Sum{L.sm[g + d], L.sl[g + d], *reinterpret_cast<const f32x4*>(&L.so[g + d][ch])});
            __syncthreads();
        }
        if (sub == 0 && rw < rows) store_row<F16>(a, jn.q0, jn.row0 + first + rw, head, ch, s.m, s.l, s.o);
    }
}

template <int D, bool F16>
__global__ __launch_bounds__(JOIN_T, 8) void paged_join_kernel(AttnArgs a, PlanArgs wide, float* wide_part, float* wide_ml, int blocks) {
    __shared__ JoinLds<D> L;
    constexpr int LG = JoinLds<D>::LG;
    const int tid = threadIdx.x;
    const int g = tid / (D / 4), ch = 4 * (tid - g * (D / 4));
    if (a.zero_tail && a.plan.cu) {
        const int64_t first = min(max(a.plan.cu[a.plan.R], 0), a.plan.T);
        const int64_t rows = (a.plan.T - first) * a.G * a.heads;       // (token, query head)
        for (int64_t r = static_cast<int64_t>(blockIdx.x) * LG + g; r < rows; r += static_cast<int64_t>(gridDim.x) * LG) {
            const int64_t t = r / (a.G * a.heads), h = r - t * (a.G * a.heads);
            if (a.zero_tail & 1) *reinterpret_cast<u32x2*>(a.out + (first + t) * a.o_t + h * a.o_h + ch) = u32x2{0, 0};
            if ((a.zero_tail & 2) && a.lse && ch == 0) a.lse[(first + t) * a.l_t + h] = -INFINITY;
        }
    }
    if (static_cast<int>(blockIdx.x) < blocks) {
        join_tiles<Narrow, D, F16>(a, L, blockIdx.x, blocks);
    } else {
        a.plan = wide;
        a.part = wide_part;
        a.ml = wide_ml;
        join_tiles<Wide, D, F16>(a, L, blockIdx.x - blocks, gridDim.x - blocks);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Sizes {
    int64_t target, wanted, most, items, joins, parts;   // most: pieces of a tile
    size_t off_counts, off_items, off_joins, off_part, off_ml, end;
};

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Where a kind's schedule and partial results lie, from `at` on.  A request's
// tiles are cut into ceil(units / per) pieces with per >= total / wanted: at
// most wanted + tiles in all, at most 2 wanted of them in tiles that are cut
// (units > per), which are at most wanted.  `tiles` bounds the tiles; short
// tables bound the pieces of one, by per >= MIN_UNITS (one 8K request on 8 key
// heads: 33 x 8 workgroups instead of 129 x 8, 14.6 us instead of 16.9).
template <typename K>
Sizes sizes_of(const hyq_paged_params& p, int64_t tiles, size_t at) {
    Sizes s{};
    s.target = std::max<int64_t>(1, K::slots(p.head_dim) / p.kv_heads);
    s.wanted = K::most(s.target, tiles);
    const int64_t keys = static_cast<int64_t>(p.max_pages) * p.page_size;
    const int64_t units = (p.window > 0 ? std::min<int64_t>(keys, static_cast<int64_t>(p.window) + K::TILE) : keys) / K::GROUP + 2;
    // pieces of a tile (no piece is shorter than MIN_UNITS, no tile cut that is hardly longer)
    s.most = units <= K::MIN_UNITS * K::UNCUT ? 1 : (units + K::MIN_UNITS - 1) / K::MIN_UNITS;
    s.items = tiles ? std::min(s.wanted + tiles, tiles * s.most) : 0;
    s.joins = s.most > 1 ? std::min(tiles, s.wanted) : 0;
    s.parts = s.joins ? std::min(s.items, 2 * s.wanted) : 0;
    s.off_counts = at;
    s.off_items = at + 256;
    s.off_joins = up256(s.off_items + s.items * sizeof(Item));
    s.off_part = up256(s.off_joins + s.joins * sizeof(Join));
    s.off_ml = up256(s.off_part + static_cast<size_t>(s.parts) * p.kv_heads * K::TILE * p.head_dim * 4);
    s.end = up256(s.off_ml + static_cast<size_t>(s.parts) * p.kv_heads * K::TILE * 2 * 4);
    return s;
}
struct Both {
    Sizes narrow, wide;
};
Both sizes_of(const hyq_paged_params& p) {
    const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.kv_repeat, R = std::min(p.num_requests, p.num_tokens);
    // without cu_seqlens every request has kv_repeat rows
    const bool narrow = p.kv_repeat <= Narrow::TILE, wide = p.cu_seqlens ? rows > Narrow::TILE : !narrow;
    Both b;
    b.narrow = sizes_of<Narrow>(p, narrow ? R : 0, 0);
    b.wide = sizes_of<Wide>(p, wide ? rows / Wide::TILE + std::min(R, rows / (Narrow::TILE + 1)) : 0, b.narrow.end);
    return b;
}

int check_pool(const char* what, size_t scale_size, int32_t head_dim, int32_t page_size, int64_t num_pages, int32_t kv_heads,
               const void* kp, const void* vp, const void* ks, const void* vs, int64_t ps_page, int64_t ps_head) {
    const std::string w = std::string(what) + ": ";
    if (head_dim != 64 && head_dim != 128) return fail(HYQ_ENOTSUP, w + "head_dim must be 64 or 128, got " + std::to_string(head_dim));
    if (!ok_page(page_size)) return fail(HYQ_ENOTSUP, w + "page_size must be a power of two from 16 to 256, got " + std::to_string(page_size));
    if (num_pages < 0 || num_pages > (int64_t{1} << 30)) return fail(HYQ_EINVAL, w + "num_pages out of range");
    if (kv_heads < 1 || kv_heads > 65535) return fail(HYQ_EINVAL, w + "key heads out of range");
    if (num_pages == 0) return HYQ_OK;
    if (!kp || !vp || !ks || !vs) return fail(HYQ_EINVAL, w + "null cache pointer");
    if (!aligned(kp, 16) || !aligned(vp, 16) || ps_page % 16 || ps_head % 16)
        return fail(HYQ_EINVAL, w + "code pages must be 16-byte aligned with strides divisible by 16");
    if (!aligned(ks, scale_size) || !aligned(vs, scale_size)) return fail(HYQ_EINVAL, w + "scales misaligned");
    return HYQ_OK;
}

// a launch has fewer than 2^32 threads along a dimension
constexpr int64_t MOST_THREADS = (int64_t{1} << 32) - 1024;
int64_t most_rows(int head_dim) { return MOST_THREADS / (head_dim / 8); }

int check_attention(const char* w, size_t scale_size, const hyq_paged_params* p) {
    if (!p) return fail(HYQ_EINVAL, std::string(w) + ": null parameters");
    const std::string s = std::string(w) + ": ";
    if (int st = check_pool(w, scale_size, p->head_dim, p->page_size, p->num_pages, p->kv_heads, p->k_pages, p->v_pages, p->k_scale,
                            p->v_scale, p->p_stride_page, p->p_stride_head))
        return st;
    if (p->kv_heads > 1024) return fail(HYQ_ENOTSUP, s + "more than 1024 key heads");   // (32-bit offsets between a row's pieces)
    if (p->kv_repeat < 1 || p->kv_repeat > 1024) return fail(HYQ_ENOTSUP, s + "kv_repeat must be 1 to 1024");
    if (p->num_requests < 0 || p->num_tokens < 0 || p->max_pages < 0 || p->window < 0)
        return fail(HYQ_EINVAL, s + "negative size");
    if (static_cast<int64_t>(p->num_tokens) * p->kv_repeat > (int64_t{1} << 26))
        return fail(HYQ_ENOTSUP, s + "more than 2^26 query rows per key head");
    if (static_cast<int64_t>(p->max_pages) * p->page_size > (int64_t{1} << 30))
        return fail(HYQ_ENOTSUP, s + "a block table row names more than 2^30 tokens");
    if (p->num_requests > (1 << 20)) return fail(HYQ_ENOTSUP, s + "more than 2^20 requests");
    if (p->dtype_fp16 != 0 && p->dtype_fp16 != 1) return fail(HYQ_EINVAL, s + "dtype_fp16 must be 0 or 1");
    if (p->zero_tail < 0 || p->zero_tail > 3) return fail(HYQ_EINVAL, s + "zero_tail must be 0 to 3");
    if (!(p->sm_scale == p->sm_scale) || std::isinf(p->sm_scale)) return fail(HYQ_EINVAL, s + "sm_scale must be finite");
    if (p->num_requests == 0 || p->num_tokens == 0) return HYQ_OK;
    if (!p->cu_seqlens && p->num_tokens != p->num_requests)
        return fail(HYQ_EINVAL, s + "without cu_seqlens every request has one token");
    if (!p->q || !p->out || !p->seq_lens || (p->max_pages > 0 && !p->block_table)) return fail(HYQ_EINVAL, s + "null pointer");
    if (!aligned(p->q, 16) || p->q_stride_t % 8 || p->q_stride_h % 8)
        return fail(HYQ_EINVAL, s + "q must be 16-byte aligned with strides divisible by 8");
    if (!aligned(p->out, 8) || p->o_stride_t % 4 || p->o_stride_h % 4)
        return fail(HYQ_EINVAL, s + "out must be 8-byte aligned with strides divisible by 4");
    if (!aligned(p->seq_lens, 4) || !aligned(p->cu_seqlens, 4) || !aligned(p->block_table, 4) || !aligned(p->lse, 4) || !aligned(p->counters, 4))
        return fail(HYQ_EINVAL, s + "lengths, table, lse and counters must be 4-byte aligned");
    const Both z = sizes_of(*p);
    if (z.wide.items * p->kv_heads > MOST_THREADS / (64 * CHUNK_WAVES))
        return fail(HYQ_ENOTSUP, s + std::to_string(z.wide.items) + " tiles of " + std::to_string(p->kv_heads) + " key heads are more than a launch holds");
    return HYQ_OK;
}

// More than 64 KiB of LDS for a kernel, once per device (`done`: a bit for each)
int raise_lds(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = uint64_t{1} << (dev & 63);
    if (e == hipSuccess && (done.load(std::memory_order_acquire) & bit)) return HYQ_OK;
    if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != hipSuccess) return fail(HYQ_EDEVICE, std::string("paged attention: LDS limit: ") + hipGetErrorString(e));
    done.fetch_or(bit, std::memory_order_release);
    return HYQ_OK;
}

// workgroups of a kind's joins, at most `most`
template <typename K, int D>
int64_t join_grid(const Sizes& s, int heads, int64_t most) {
    return std::min<int64_t>(s.joins * heads * (K::TILE / K::join_rows(JOIN_T / (D / 4))), most);
}

// KERNELS: a cache's narrow and chunk kernels and the chunk kernel's LDS
template <int D, bool F16, typename KERNELS>
int launch_attention(const char* what, AttnArgs a, const PlanArgs& narrow, const PlanArgs& wide, const Both& s, char* ws, hipStream_t st) {
    auto partials = [&](const Sizes& z) {
        a.part = reinterpret_cast<float*>(ws + z.off_part);
        a.ml = reinterpret_cast<float*>(ws + z.off_ml);
    };
    if (s.wide.items) {
        a.plan = wide;
        partials(s.wide);
        static std::atomic<uint64_t> raised{0};
        if (int rc = raise_lds(reinterpret_cast<const void*>(KERNELS::chunk), KERNELS::chunk_lds, raised)) return rc;
        KERNELS::chunk<<<dim3(static_cast<unsigned>(s.wide.items * a.heads)), dim3(64 * CHUNK_WAVES), KERNELS::chunk_lds, st>>>(a);
    }
    a.plan = narrow;
    partials(s.narrow);
    if (s.narrow.items) KERNELS::narrow(a)<<<dim3(static_cast<unsigned>(s.narrow.items), a.heads), dim3(64 * WAVES), 0, st>>>(a);
    // a round of resident workgroups (two a CU) for the kind that there is, half
    // of one each where both may be
    const int64_t most = s.narrow.joins && s.wide.joins ? 256 : 512;
    int64_t jn = a.counters ? 0 : join_grid<Narrow, D>(s.narrow, a.heads, most);
    const int64_t jw = join_grid<Wide, D>(s.wide, a.heads, most);
    if (a.zero_tail && a.plan.cu && jn + jw == 0) jn = 1;
    if (jn + jw)
        paged_join_kernel<D, F16><<<dim3(static_cast<unsigned>(jn + jw)), dim3(JOIN_T), 0, st>>>(
            a, wide, reinterpret_cast<float*>(ws + s.wide.off_part), reinterpret_cast<float*>(ws + s.wide.off_ml), static_cast<int>(jn));
    return check_launch(what);
}

// Whether the attention launch joins the pieces itself: a decode step (a ragged
// call's join launch also clears rows) with counters, in no captured graph, whose
// replays on another stream would share them.  One 8K sequence takes 12.0 us
// instead of 14.1, 200 requests 29.0 instead of 31.2, one of 1K 10.5 instead of
// 13.1; but where a request may be cut into more than 48 pieces, one workgroup
// takes longer than the launch does (one 32K sequence 22.9, 20.5).
bool join_here(const hyq_paged_params& p, const Both& s, hipStream_t st) {
    if (!p.counters || p.cu_seqlens || s.wide.items || s.narrow.joins * p.kv_heads * COUNTER_PAD * 2 > HYQ_PAGED_COUNTERS) return false;
    if (!aligned(p.counters, 8) || st == hipStreamPerThread) return false;     // (that handle names a stream of every thread)
    if (s.narrow.most > 48 && s.narrow.wanted > 48 * static_cast<int64_t>(p.num_requests)) return false;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &status) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return status == hipStreamCaptureStatusNone;
}

size_t attention_workspace(const char* what, size_t scale_size, const hyq_paged_params* p) {
    if (check_attention(what, scale_size, p) != HYQ_OK || p->num_requests == 0 || p->num_tokens == 0) return 0;
    return sizes_of(*p).wide.end;
}

template <template <int, bool> class KERNELS>
int attention(const char* what, size_t scale_size, const hyq_paged_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = check_attention(what, scale_size, p)) return st;
    if (p->num_requests == 0 || p->num_tokens == 0) return HYQ_OK;
    const Both s = sizes_of(*p);
    if (!workspace || workspace_bytes < s.wide.end)
        return fail(HYQ_ENOSPC, std::string(what) + ": workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(s.wide.end) + " needed");
    if (!aligned(workspace, 256)) return fail(HYQ_EINVAL, std::string(what) + ": workspace must be 256-byte aligned");
    char* ws = static_cast<char*>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    // no table row names 2^30 tokens: such a window hides nothing, and position -
    // window stays within 32 bits also for tokens before position 0
    const int32_t window = p->window < (1 << 30) ? p->window : 0;
    auto plan_of = [&](const Sizes& z) {
        return PlanArgs{p->seq_lens, p->cu_seqlens, p->num_requests, p->num_tokens, p->kv_repeat, window, p->max_pages * p->page_size,
                        static_cast<int32_t>(z.target), static_cast<int32_t>(z.items),
                        static_cast<int32_t>(z.parts), static_cast<int32_t>(z.joins), reinterpret_cast<Counts*>(ws + z.off_counts),
                        reinterpret_cast<Item*>(ws + z.off_items), reinterpret_cast<Join*>(ws + z.off_joins)};
    };
    const PlanArgs narrow = plan_of(s.narrow), wide = plan_of(s.wide);
    if (p->num_requests > INLINE_R) paged_plan_kernel<<<dim3(s.wide.items ? 2 : 1), dim3(PLAN_T), 0, st>>>(narrow, wide);
    const bool here = join_here(*p, s, st);
    std::unique_lock<std::mutex> lock(call_order().mutex, std::defer_lock);
    if (here) lock.lock();
    const uint64_t call = here ? ++call_order().calls : 0;
    const AttnArgs a{static_cast<const uint16_t*>(p->q), p->q_stride_t, p->q_stride_h, static_cast<uint16_t*>(p->out), p->o_stride_t, p->o_stride_h,
                     p->lse, static_cast<int64_t>(p->kv_heads) * p->kv_repeat, p->k_pages, p->v_pages, p->p_stride_page, p->p_stride_head,
                     p->k_scale, p->v_scale, p->s_stride_page, p->s_stride_head, p->block_table, p->bt_stride, narrow, nullptr, nullptr,
                     here ? reinterpret_cast<uint64_t*>(p->counters) : nullptr, call << CALL_SHIFT, p->kv_repeat, p->kv_heads, log2i(p->page_size), static_cast<int32_t>(p->num_pages), window, p->zero_tail,
                     p->sm_scale * 1.44269504f};
    if (p->head_dim == 128)
        return p->dtype_fp16 ? launch_attention<128, true, KERNELS<128, true>>(what, a, narrow, wide, s, ws, st)
                             : launch_attention<128, false, KERNELS<128, false>>(what, a, narrow, wide, s, ws, st);
    return p->dtype_fp16 ? launch_attention<64, true, KERNELS<64, true>>(what, a, narrow, wide, s, ws, st)
                         : launch_attention<64, false, KERNELS<64, false>>(what, a, narrow, wide, s, ws, st);
}

}  // namespace
}  // namespace hyq
