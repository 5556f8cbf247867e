// The paged 4-bit KV cache: batch layout, append, read-back and attention
// over block tables.
//
// Cache: int8 [pages, key heads, page, D/2] codes of hyq_quant_pack's 4-bit
// format (the even channel in the low nibble) and fp16 [pages, key heads,
// page] scales, K and V alike; token j of request r sits in page
// block_table[r][j / page] at row j % page.  Pages are a power of two of 16
// to 256 tokens, so a 16-token tile never crosses a page and every tile's
// rows are one base address plus 32-bit lane offsets; bases are 64-bit.
#include "hyq_common.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <string>

namespace hyq {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int MAX_REQUESTS = 16384;      // two int32 prefix arrays of a batch fit in LDS
constexpr int MIN_PAGE = 16, MAX_PAGE = 256;

bool ok_page(int page) { return page >= MIN_PAGE && page <= MAX_PAGE && (page & (page - 1)) == 0; }
int log2i(int x) {
    int l = 0;
    while ((1 << l) < x) ++l;
    return l;
}

// ---------------------------------------------------------------------------
// batch layout
// ---------------------------------------------------------------------------
// cu = prefix sums of the new tokens, first = prefix sums of the pages that
// each request takes, ceil(len / page) - ceil(ctx / page); token t of request
// r has position ctx_r + t - cu_r.  Every workgroup scans the R lengths by
// itself (they stay in the L2) and keeps both prefix arrays in LDS, so the
// layout is one launch; token and page entries then find their request by a
// binary search.  A new page's id comes from the free list, never from the
// table entry another workgroup writes.  Bound by the chain lengths -> scan ->
// search -> table -> store, not by bytes: 3.7 us for 24 requests, 5.2 us for
// 1000 requests and 150000 tokens (2.4 MB), both in a captured graph.  512
// threads with two requests each and 512 tokens a workgroup are the best of
// what was measured there: 256 threads and 1024 tokens 7.7 us, 1024 threads
// 5.9, 2048 tokens 11.0.
constexpr int BT = 512;                  // threads
constexpr int PER = 2;                   // requests per thread and round of the scan
constexpr int BATCH_TOKENS = 512;        // tokens per workgroup

struct BatchArgs {
    const int32_t* ctx;
    const int32_t* fresh;
    int32_t* table;
    int64_t bt_stride;
    const int32_t* free_pages;
    int32_t *cu, *lens, *used;
    int64_t *slots, *positions;
    int32_t R, max_pages, num_free, page_log2, tokens;
};

__device__ __forceinline__ int ceil_pages(int tokens, int page_log2) {
    return static_cast<int>((static_cast<uint32_t>(tokens) + (1u << page_log2) - 1u) >> page_log2);
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

__global__ __launch_bounds__(BT) void paged_batch_kernel(BatchArgs a) {
    extern __shared__ int32_t lds[];
    int32_t* const cu = lds;                       // [R + 1]
    int32_t* const first = lds + a.R + 1;          // [R + 1]
    __shared__ int32_t wsum[2][BT / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int base_t = 0, base_p = 0;
    for (int r0 = 0; r0 < a.R; r0 += BT * PER) {
        const int r = r0 + tid * PER;    // this thread's requests: r .. r + PER - 1
        int n[PER], p[PER], st = 0, sp = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool in = r + j < a.R;
            const int c = in ? max(a.ctx[r + j], 0) : 0;
            n[j] = in ? max(a.fresh[r + j], 0) : 0;
            p[j] = ceil_pages(c + n[j], a.page_log2) - ceil_pages(c, a.page_log2);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) { st += n[j]; sp += p[j]; }
        const int it = scan_dpp(st), ip = scan_dpp(sp);
        if (lane == 63) { wsum[0][w] = it; wsum[1][w] = ip; }
        __syncthreads();
        int bt = base_t + it - st, bp = base_p + ip - sp;
#pragma unroll
        for (int i = 0; i < BT / 64; ++i) {
            if (i < w) { bt += wsum[0][i]; bp += wsum[1][i]; }
            base_t += wsum[0][i];
            base_p += wsum[1][i];
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (r + j < a.R) { cu[r + j] = bt; first[r + j] = bp; }
            bt += n[j];
            bp += p[j];
        }
        if (r0 + BT * PER < a.R) __syncthreads();
    }
    if (tid == 0) { cu[a.R] = base_t; first[a.R] = base_p; }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int r = tid; r <= a.R; r += BT) {
            a.cu[r] = cu[r];
            if (r < a.R) a.lens[r] = max(a.ctx[r], 0) + max(a.fresh[r], 0);
        }
        if (tid == 0) a.used[0] = base_p;
    }
    // the pages taken: entry i of the free list goes to request r at table
    // column ceil(ctx / page) + i - first[r].  (Both loops count without a sign:
    // a step past a count below 2^31 does not wrap.)
    const uint32_t start = blockIdx.x * BT + tid, stride = gridDim.x * BT;
    for (uint32_t u = start; u < static_cast<uint32_t>(max(base_p, 0)); u += stride) {
        const int i = static_cast<int>(u);
        const int r = last_at_most(first, a.R - 1, i);
        const int col = ceil_pages(max(a.ctx[r], 0), a.page_log2) + i - first[r];
        if (static_cast<uint32_t>(col) < static_cast<uint32_t>(a.max_pages))
            a.table[r * a.bt_stride + col] = i < a.num_free ? a.free_pages[i] : -1;
    }
    const int page = 1 << a.page_log2;
    for (uint32_t u = start; u < static_cast<uint32_t>(a.tokens); u += stride) {
        const int t = static_cast<int>(u);
        int64_t slot = -1, pos = -1;
        if (t < base_t) {
            const int r = last_at_most(cu, a.R - 1, t);
            const int c = max(a.ctx[r], 0);
            const int x = c + t - cu[r];
            const int col = x >> a.page_log2, old = ceil_pages(c, a.page_log2);
            int id = -1;
            if (static_cast<uint32_t>(col) < static_cast<uint32_t>(a.max_pages)) {
                const int i = first[r] + col - old;
                id = col < old ? a.table[r * a.bt_stride + col]
                     : static_cast<uint32_t>(i) < static_cast<uint32_t>(a.num_free) ? a.free_pages[i] : -1;
            }
            pos = x;
            if (id >= 0) slot = (static_cast<int64_t>(id) << a.page_log2) + (x & (page - 1));
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
}

// ---------------------------------------------------------------------------
// append and read back
// ---------------------------------------------------------------------------
struct RowArgs {
    const uint16_t *k, *v;               // [tokens, key heads, D]
    int64_t kt, kh, vt, vh;
    uint16_t *ok, *ov;                   // the read-back's rows, contiguous
    const int64_t* slots;
    int8_t *kp, *vp;
    int64_t ps_page, ps_head;
    uint16_t *ks, *vs;
    int64_t ss_page, ss_head;
    int64_t num_slots;
    uint32_t rows, heads;                // rows = tokens * heads
    int32_t page_log2, lpt_log2;
};

// max over each aligned group of 8 lanes, or of 16
__device__ __forceinline__ float max_lanes(float v, bool sixteen) {
    auto dpp = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v = fmaxf(v, dpp(v, std::integral_constant<int, 0xb1>{}));    // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp(v, std::integral_constant<int, 0x4e>{}));    // quad_perm [2,3,0,1]
    v = fmaxf(v, dpp(v, std::integral_constant<int, 0x141>{}));   // row_half_mirror
    if (sixteen) v = fmaxf(v, dpp(v, std::integral_constant<int, 0x140>{}));   // row_mirror
    return v;
}

// hyq_quant_pack's 4-bit rows (quant_row_codes) into their slots: D/8 lanes
// of 8 channels own a row, blockIdx.y picks K or V, one launch for both.
// HBM-bound: 2D bytes read and D/2 + 2 written per row.  8192 tokens of 8 heads
// of 128 (42 MB) take 10.5 us, 4.0 TB/s with the launch's 2.5 us in it; one row
// per thread, since two or four change nothing there (20.2 us with the read-back
// for 1 and 2, 20.5 for 4) and cost latency at 16 tokens (4.6 us against 5.0 and
// 5.9).
template <bool F16>
__global__ __launch_bounds__(256) void paged_append_kernel(RowArgs a) {
    const int lpt = 1 << a.lpt_log2, sub = threadIdx.x & (lpt - 1);
    const uint32_t row = blockIdx.x * (256u >> a.lpt_log2) + (threadIdx.x >> a.lpt_log2);
    const bool is_v = blockIdx.y != 0;
    const uint32_t rr = row < a.rows ? row : a.rows - 1;
    const uint32_t t = rr / a.heads, h = rr - t * a.heads;
    const uint16_t* src = is_v ? a.v + t * a.vt + h * a.vh : a.k + t * a.kt + h * a.kh;
    const int64_t slot = a.slots[t];
    const uint4 raw = reinterpret_cast<const uint4*>(src)[sub];
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (F16) {
            x[2 * i] = f16_bits_to_f32(static_cast<uint16_t>(w[i]));
            x[2 * i + 1] = f16_bits_to_f32(static_cast<uint16_t>(w[i] >> 16));
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(max_lanes(amax, lpt > 8), 1e-5f);
    _Float16 s16;
    uint32_t c[8];
    quant_row_codes<4>(x, amax, s16, c);
    if (row >= a.rows || slot < 0 || slot >= a.num_slots) return;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= (c[i] & 15u) << (4 * i);
    const int64_t page = slot >> a.page_log2, off = slot & ((1 << a.page_log2) - 1);
    int8_t* dst = (is_v ? a.vp : a.kp) + page * a.ps_page + h * a.ps_head + ((off * 4) << a.lpt_log2);
    reinterpret_cast<uint32_t*>(dst)[sub] = word;
    if (sub == 0) (is_v ? a.vs : a.ks)[page * a.ss_page + h * a.ss_head + off] = __builtin_bit_cast(uint16_t, s16);
}

// Rows of the cache by slot as bf16 or fp16 values, code * scale rounded once
// (the product is exact in fp32); slots outside the pool give zero rows.
// HBM-bound: D/2 + 2 bytes read and 2D written per row; 8192 tokens of 8 heads of
// 128 (42 MB) take 9.6 us, 4.4 TB/s.
template <bool F16>
__global__ __launch_bounds__(256) void paged_gather_kernel(RowArgs a) {
    const int lpt = 1 << a.lpt_log2, sub = threadIdx.x & (lpt - 1);
    const uint32_t row = blockIdx.x * (256u >> a.lpt_log2) + (threadIdx.x >> a.lpt_log2);
    if (row >= a.rows) return;
    const bool is_v = blockIdx.y != 0;
    const uint32_t t = row / a.heads, h = row - t * a.heads;
    const int64_t slot = a.slots[t];
    uint32_t o[4] = {0, 0, 0, 0};
    if (slot >= 0 && slot < a.num_slots) {
        const int64_t page = slot >> a.page_log2, off = slot & ((1 << a.page_log2) - 1);
        const int8_t* src = (is_v ? a.vp : a.kp) + page * a.ps_page + h * a.ps_head + ((off * 4) << a.lpt_log2);
        const uint32_t word = reinterpret_cast<const uint32_t*>(src)[sub];
        const float s = f16_bits_to_f32((is_v ? a.vs : a.ks)[page * a.ss_page + h * a.ss_head + off]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = static_cast<float>(static_cast<int>(word << (28 - 8 * i)) >> 28) * s;
            const float hi = static_cast<float>(static_cast<int>(word << (24 - 8 * i)) >> 28) * s;
            o[i] = F16 ? f32_to_f16_bits(lo) | (static_cast<uint32_t>(f32_to_f16_bits(hi)) << 16) : pack_bf16x2(lo, hi);
        }
    }
    reinterpret_cast<uint4*>((is_v ? a.ov : a.ok) + (static_cast<int64_t>(row) * 8 << a.lpt_log2))[sub] =
        make_uint4(o[0], o[1], o[2], o[3]);
}

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
__device__ __forceinline__ uint32_t nib2(uint32_t x, int s, uint32_t magic) { return ((x >> s) & 0x000f000fu) ^ magic; }
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
template <int I>
__device__ __forceinline__ float quad_bcast(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), I * 0x55, 0xf, 0xf, true));
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

// ---------------------------------------------------------------------------
// attention: 16 query rows per workgroup
// ---------------------------------------------------------------------------
struct AttnArgs {
    const uint16_t* q;
    int64_t q_t, q_h;
    uint16_t* out;
    int64_t o_t, o_h;
    float* lse;
    int64_t l_t;
    const int8_t *kp, *vp;
    int64_t ps_page, ps_head;
    const uint16_t *ks, *vs;
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

// A workgroup has one KV head of a tile of 16 rows (a request's tokens times the
// G query heads) and a range of keys; its four wavefronts take every fourth
// 32-key step and join through LDS at the end.
//   QK  S^T[key][row] = K . Q^T with v_mfma_f32_16x16x32_f16.  A K operand is the
//       code's offset form u = code + 8 as the fp16 subnormal u 2^-24, two bit
//       operations per pair of codes; the accumulators start at -8 sum(q) 2^-24,
//       so that the score is exact but for fp32 roundings.
//   softmax: a row's maximum moves only when a score passes it by SLACK (its own
//       scores alone move it), sums in fp32.
//   PV  O^T[channel][row] = V^T . P'^T with v_mfma_f32_16x16x32_bf16, V operands
//       the bf16 numbers 128 + u, P' = p v_scale as the sum of two bf16 numbers
//       (2^-16 of a weight is lost; one bf16 number, 2^-8, made a bf16 output's
//       error 2.4e-3 where its own rounding is 1.7e-3, and was 3 to 6% faster):
//       136 sum(P') is taken off every 96 keys of a wavefront, from the same
//       rounded P' by products with ones.  The running sum carries up to 140
//       times those keys' weights, and its fp32 roundings stay in the result:
//       taken off at the end alone they made a relative error of 2.4e-3 over 32K
//       keys in one piece, where an fp16 output's own rounding is 2.1e-4 (1% of
//       the time).  Outputs of either type are then as good as their type.
// Bound by the cache's bytes: 16 requests of 32K keys (554 MB) take 103 to 106
// us, 5.3 TB/s where a copy reaches 5.1 and a stream of reads 6.8.  What feeds it is the
// ring of three groups' loads in registers per wavefront (two: 121 us), no LDS
// on the way in, and 3 resident workgroups a CU.  Short calls are bound by the
// chain lengths -> table -> rows -> pieces: 12.0 us for one request of 8K keys.
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

template <int D>
struct Raw {
    uint32_t k[2][D / 32];               // tile t: row c's channels (D/4) kb .. of token 16t + 4(c & 3) + (c >> 2)
    uint32_t v[8];                       // slot e: token 4e + kb, 8 channels
    uint32_t sk[2], sv[2];               // tile t: scale bits of token 16t + 4(c & 3) + kb
    int first;                           // first token of the group
    int ok;                              // bit t: tile t's page is inside the pool
};

template <int D, bool F16>
__global__ __launch_bounds__(64 * WAVES, D == 64 ? 4 : 3) void paged_attn_kernel(AttnArgs a) {
    constexpr int TILE = Narrow::TILE, GROUP = Narrow::GROUP;
    constexpr int NB = D / 16;           // PV products per group
    constexpr int KW = D / 32;           // QK products (and K dwords) per tile
    constexpr int ROWB = D / 2;          // packed bytes per token
    __shared__ float red[WAVES][TILE][D + 4];
    __shared__ float redm[WAVES][TILE], redl[WAVES][TILE];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int head = blockIdx.y;
    Item it;
    if (!find_item<Narrow>(a.plan, blockIdx.x, head, lane, it)) return;
    const int c = lane & 15, kb = lane >> 4;
    const int nrows = min(TILE, it.qlen * a.G - it.row0);

    // ---- the first loads: queries, page ids, then the first groups' rows ----
    // (a decode step's tile is its one token's G rows: no division by G)
    const bool one = it.qlen == 1;
    const int row = it.row0 + min(c, nrows - 1);
    const int tok = one ? 0 : row / a.G, hq = row - tok * a.G;
    const uint16_t* qp = a.q + (static_cast<int64_t>(it.q0) + tok) * a.q_t + (static_cast<int64_t>(head) * a.G + hq) * a.q_h + (D / 4) * kb;
    const int32_t* trow = a.table + it.req * a.bt_stride;
    const int steps = (max(it.key1 - it.key0, 0) + GROUP - 1) / GROUP;
    const int mine = steps > w && a.num_pages > 0 ? (steps - w + WAVES - 1) / WAVES : 0;   // this wavefront's groups w, w + 4, ...
    // page ids of this wavefront's next 32 groups, tile t of group i in lane 2i + t
    auto ids_at = [&](int i0) -> int {
        const int t = it.key0 + GROUP * (w + WAVES * (i0 + (lane >> 1))) + 16 * (lane & 1);
        return trow[min(t, it.key1 - 1) >> a.page_log2];
    };
    int ids = 0, ids_next = 0;
    if (mine > 0) ids = ids_at(0);
    if (mine > 32) ids_next = ids_at(32);
    u32x4 qr[KW];
#pragma unroll
    for (int m = 0; m < KW; ++m) qr[m] = *reinterpret_cast<const u32x4*>(qp + 8 * m);

    const int64_t hk = head * a.ps_head, hs = head * a.ss_head;
    const int page_mask = (1 << a.page_log2) - 1;
    const uint32_t klane = (4 * (c & 3) + (c >> 2)) * ROWB + (ROWB / 4) * kb;
    const uint32_t vlane = kb * ROWB + (D == 128 ? 4 * c : 4 * (c & 7));
    const uint32_t slane = (4 * (c & 3) + kb) * 2;
    // Every load goes through a buffer descriptor over its 16-token tile, of
    // range 0 past this wavefront's groups or where the page is not in the
    // pool: such loads give zeros and touch no memory, so the ring's loads are
    // unconditional and their wait counts exact.
    auto load = [&](Raw<D>& r, int i) {
        if (i > 0 && (i & 31) == 0) {
            ids = ids_next;
            ids_next = mine > i + 32 ? ids_at(i + 32) : 0;
        }
        r.first = it.key0 + GROUP * (w + WAVES * i);
        r.ok = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int id = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + t);
            const bool ok = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_pages);
            const bool in = ok && i < mine;
            r.ok |= ok ? 1 << t : 0;
            const int64_t pg = ok ? id : 0;
            const int t0 = (min(r.first + 16 * t, it.key1 - 1) & page_mask) & ~15;
            const int64_t co = pg * a.ps_page + hk + t0 * ROWB, so = pg * a.ss_page + hs + t0;
            const Rsrc rk = make_rsrc(a.kp + co, in ? 16 * ROWB : 0), rv = make_rsrc(a.vp + co, in ? 16 * ROWB : 0);
            const Rsrc rks = make_rsrc(a.ks + so, in ? 32 : 0), rvs = make_rsrc(a.vs + so, in ? 32 : 0);
            if constexpr (D == 128) {
                const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, klane, 0, NT));
                r.k[t][0] = x[0]; r.k[t][1] = x[1]; r.k[t][2] = x[2]; r.k[t][3] = x[3];
            } else {
                const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, klane, 0, NT));
                r.k[t][0] = x[0]; r.k[t][1] = x[1];
            }
            r.sk[t] = __builtin_amdgcn_raw_buffer_load_b16(rks, slane, 0, 0);
            r.sv[t] = __builtin_amdgcn_raw_buffer_load_b16(rvs, slane, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) r.v[4 * t + e] = __builtin_amdgcn_raw_buffer_load_b32(rv, vlane + 4 * e * ROWB, 0, NT);
        }
    };
    Raw<D> ring[3];
    load(ring[0], 0);
    load(ring[1], 1);

    // ---- queries: B operands, row c's channels (D/4) kb + 8m + [0,4,1,5,2,6,3,7] ----
    float amax = 0.f;
#pragma unroll
    for (int m = 0; m < KW; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(half_at<F16>(qr[m][i], 0)), fabsf(half_at<F16>(qr[m][i], 1))));
    // (a power of two of each row's own: rows of any magnitude stand side by side)
    amax = col_max(amax);
    if (!(amax < INFINITY)) amax = 0.f;
    const int qe = q_exponent(amax);
    const float qs = pow2(-qe), row_scale = pow2(qe);
    f16x8 qop[KW];
#pragma unroll
    for (int m = 0; m < KW; ++m) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = half_at<F16>(qr[m][i >> 1], i & 1) * qs;
        qop[m] = f16x8{static_cast<_Float16>(f[0]), static_cast<_Float16>(f[4]), static_cast<_Float16>(f[1]), static_cast<_Float16>(f[5]),
                       static_cast<_Float16>(f[2]), static_cast<_Float16>(f[6]), static_cast<_Float16>(f[3]), static_cast<_Float16>(f[7])};
    }
    const float qk = a.scale * 16777216.0f;                // K operands are codes * 2^-24
    f32x4 kbias = {0.f, 0.f, 0.f, 0.f};
    {
        const u32x4 half = {0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u};
#pragma unroll
        for (int m = 0; m < KW; ++m) kbias = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, half), qop[m], kbias, 0, 0, 0);
        kbias = -kbias;
    }
    // this lane's row sees the keys [lo, hi]
    const int pos = it.len - it.qlen + tok;
    const int lo = first_key(pos, a.window), hi = pos;
    const int tok0 = one ? 0 : it.row0 / a.G, tok1 = one ? 0 : (it.row0 + nrows - 1) / a.G;
    const int all_hi = it.len - it.qlen + tok0;                             // every row sees keys up to here
    const int all_lo = first_key(it.len - it.qlen + tok1, a.window);        // and from here

    float m_run = M_INIT, l_run = 0.f;
    f32x4 acc[NB], ones = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](const Raw<D>& r) {
        float s[8];
        const float sk[2] = {f16_bits_to_f32(static_cast<uint16_t>(r.sk[0])) * qk, f16_bits_to_f32(static_cast<uint16_t>(r.sk[1])) * qk};
        const float sv[2] = {f16_bits_to_f32(static_cast<uint16_t>(r.sv[0])), f16_bits_to_f32(static_cast<uint16_t>(r.sv[1]))};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 x = kbias;
#pragma unroll
            for (int m = 0; m < KW; ++m) {
                const uint32_t kw = r.k[t][m];
                const u32x4 o = {nib2(kw, 0, 0x00080008u), nib2(kw, 4, 0x00080008u), nib2(kw, 8, 0x00080008u), nib2(kw, 12, 0x00080008u)};
                x = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, o), qop[m], x, 0, 0, 0);
            }
            s[4 * t + 0] = x[0] * quad_bcast<0>(sk[t]);
            s[4 * t + 1] = x[1] * quad_bcast<1>(sk[t]);
            s[4 * t + 2] = x[2] * quad_bcast<2>(sk[t]);
            s[4 * t + 3] = x[3] * quad_bcast<3>(sk[t]);
        }
        // masked keys: behind the row's own position or before its window,
        // past the piece, or in a page outside the pool.  Their scores and
        // their P' are selected, not multiplied away: the scales there may be
        // anything.
        uint32_t dead = 0;
        const bool edge = r.first + GROUP - 1 > min(all_hi, it.key1 - 1) || r.first < all_lo || r.ok != 3;
        if (edge) {
            const int top = min(hi, it.key1 - 1);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = r.first + 4 * e + kb;
                if (j > top || j < lo || !((r.ok >> (e >> 2)) & 1)) {
                    s[e] = -INFINITY;
                    dead |= 1u << e;
                }
            }
        }
        float mx = vmax3(s[0], s[1], s[2]);
        mx = vmax3(mx, s[3], s[4]);
        mx = vmax3(mx, s[5], s[6]);
        mx = vmax2(mx, s[7]) * row_scale;
        if (__builtin_amdgcn_ballot_w64(mx > m_run + SLACK)) {
            mx = col_max(mx);
            const float mnew = mx > m_run + SLACK ? mx : m_run;        // (a row's own scores alone move its maximum)
            const float alpha = fast_exp2(m_run - mnew);
            l_run *= alpha;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) acc[nb] *= alpha;
            ones *= alpha;
            m_run = mnew;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[e] = fast_exp2(__builtin_fmaf(s[e], row_scale, -m_run));
            l_run += s[e];
        }
        float p[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            p[4 * t + 0] = s[4 * t + 0] * quad_bcast<0>(sv[t]);
            p[4 * t + 1] = s[4 * t + 1] * quad_bcast<1>(sv[t]);
            p[4 * t + 2] = s[4 * t + 2] * quad_bcast<2>(sv[t]);
            p[4 * t + 3] = s[4 * t + 3] * quad_bcast<3>(sv[t]);
        }
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = (dead >> e) & 1 ? 0.f : p[e];
        }
        const u32x4 pw = {pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
        const bf16x8 pop = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] -= half_at<false>(pw[i >> 1], i & 1);
        const u32x4 pl = {pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
        const bf16x8 plo = __builtin_bit_cast(bf16x8, pl);
        uint32_t vlo[4], vhi[4];
#pragma unroll
        for (int pr = 0; pr < 4; ++pr) {
            uint32_t x = r.v[2 * pr], y = r.v[2 * pr + 1];
            if constexpr (D == 64) {     // rows 8..15 of a product are the upper four channels of a dword
                x = c >= 8 ? x >> 16 : x;
                y = c >= 8 ? y >> 16 : y;
            }
            vlo[pr] = perm(y, x, 0x05040100u);
            vhi[pr] = perm(y, x, 0x07060302u);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const uint32_t* src = nb < 4 ? vlo : vhi;
            const int sh = 4 * (nb & 3);
            const u32x4 o = {nib2(src[0], sh, 0x43084308u), nib2(src[1], sh, 0x43084308u), nib2(src[2], sh, 0x43084308u), nib2(src[3], sh, 0x43084308u)};
            acc[nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o), pop, acc[nb], 0, 0, 0);
            acc[nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o), plo, acc[nb], 0, 0, 0);
        }
        const u32x4 onesw = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
        ones = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, onesw), pop, ones, 0, 0, 0);
        ones = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, onesw), plo, ones, 0, 0, 0);
    };
    for (int i = 0; i < mine; i += 3) {
        load(ring[2], i + 2);
        compute(ring[0]);
        load(ring[0], i + 3);
        if (i + 1 < mine) compute(ring[1]);
        load(ring[1], i + 4);
        if (i + 2 < mine) compute(ring[2]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)  // the codes' offset
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[nb][j] = __builtin_fmaf(-136.0f, ones[j], acc[nb][j]);
        ones = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- the four wavefronts' results, joined through LDS ----
    l_run = col_sum(l_run);
    if (kb == 0) { redm[w][c] = m_run; redl[w][c] = l_run; }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 4 * kb + i;
            const int ch = D == 128 ? 8 * j + nb : 8 * (j & 7) + 4 * (j >> 3) + nb;
            red[w][c][ch] = acc[nb][i];
        }
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

// ---------------------------------------------------------------------------
// attention: CHUNK query rows per workgroup
// ---------------------------------------------------------------------------
// A wavefront owns 32 rows.  The codes of 64 keys at a time are turned into
// fp16 operands once for all rows of the workgroup and laid in LDS, two blocks
// ahead of the products.
//   QK  S^T[key][row] = K . Q^T  with v_mfma_f32_32x32x16_f16; codes and (scaled
//       by a power of two) queries are exact, the K scale multiplies the fp32
//       score in the fma that subtracts the reference: t = S k_scale - M.
//   PV  O^T[channel][row] = V^T . P'^T, P' = fp16(2^t v_scale) against the exact
//       codes, V^T by transposing LDS reads.  The reference M of a row follows
//       max(score) + log2 of the largest V scale of 16 keys, so that P' keeps to
//       [0, 2^13]; rounding P' to 11 bits once is the only rounding between the
//       scores and the output.  Where the 16 scales do not lie within a factor of
//       2^9, the largest may be another key's than the largest score's, and M so
//       high that P' sinks below fp16's 2^-14: there M follows max(score + log2 V
//       scale), key by key.
// Bound by the matrix pipe and the VALU work that has to run beside it: 2048
// tokens at 8192 (309 GFLOP) take 353 to 377 us by box, 0.82 to 0.87 PFLOP/s where a large matrix
// product reaches 1.35, and the products with their LDS reads alone take 226 us.
// So the block is worked on in halves of 32 keys: the scores of one half run
// beside the weights of the half before, and the first four wavefronts have
// priority, so that the two of a SIMD do not wait for the same pipe (without
// halves 437 us).  Rows are padded instead of swizzled: operand addresses are
// constants then (swizzled 437).  256 rows per workgroup, since a block's
// conversion is paid once per tile (16-row wavefronts, four a SIMD: 421 at best).
// Output register i of a lane (row l & 31, half h = l >> 5) of a 32-key product
// is key 8 (i >> 2) + 4 h + (i & 3); registers 8s .. 8s + 7 are the B operand of
// step s of P.V, without a shuffle.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
constexpr float P_SHIFT = 6.0f;          // P' is at most 2^(P_SHIFT + SLACK_W + 1)
constexpr float SLACK_W = 6.0f;
constexpr int BLK = 64;                  // keys per block
constexpr int BUFS = 3;                  // blocks in LDS
constexpr float BAD = 4096.0f;
constexpr float FAR = 8.0f;              // binary orders that the V scales of 16 keys may span

__device__ __forceinline__ uint32_t pk_sub1032(uint32_t x) {
    const f16x2 b = {static_cast<_Float16>(1032.0f), static_cast<_Float16>(1032.0f)};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - b);
}
// two codes of a word as fp16: 1024 + (nibble ^ 8) is exact, so is minus 1032
__device__ __forceinline__ uint32_t codes2(uint32_t x, int s) { return pk_sub1032(nib2(x, s, 0x64086408u)); }
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
    const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}

// Bytes from a key's row of D fp16 channels to the next's.  16 lanes of a K
// operand read (neighbouring rows, one 16-byte chunk) and 32 of a transposing V
// read (4 rows, 64 bytes) fall on all 64 banks once by the padding, so a lane's
// operands are one address and constants.
template <int D> constexpr int KROW = 2 * D + 16;
template <int D> constexpr int VROW = 2 * D + 64;

template <int D>
struct ChunkLds {
    uint8_t k[BUFS][BLK * KROW<D>];
    uint8_t v[BUFS][BLK * VROW<D>];
    float ks[BUFS][BLK];                 // K scale * qk
    float vs[BUFS][BLK];                 // V scale, 0 where it is not finite or not to be looked at
    float ve[BUFS][4];                   // per 16-key tile: log2 bound of vs, BAD more if the keys need care
    uint32_t care[BUFS][4];              // bits 0..15: keys whose V scale is not finite; bit 16: the page is in the pool
    float red[2][CHUNK_WAVES];
};

// e with x < 2^e, x >= 0 finite (an fp16 value: at least 2^-24, or 0, which takes
// a bound so low that it does not count beside others, and that 2^30 weights of
// 2^(12 + 79) do not overflow)
__device__ __forceinline__ float scale_bound(float x) {
    return static_cast<float>(__builtin_amdgcn_frexp_expf(fmaxf(x, 0x1p-80f)));
}

template <int D, bool F16>
__global__ __launch_bounds__(64 * CHUNK_WAVES, 2) void paged_chunk_kernel(AttnArgs a) {
    constexpr int KM = D / 16;           // QK products per 32 keys
    constexpr int DT = D / 32;           // 32-channel tiles of V
    constexpr int ROWB = D / 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    ChunkLds<D>& L = *reinterpret_cast<ChunkLds<D>*>(lds_raw);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int head = blockIdx.x % a.heads;
    Item it;
    if (!find_item<Wide>(a.plan, blockIdx.x / a.heads, head, lane, it)) return;
    const int r32 = lane & 31, h = lane >> 5;
    const int nrows = min(CHUNK, it.qlen * a.G - it.row0);

    // ---- queries ----
    const int rt = 32 * w + r32;                          // row within the tile (behind its last: that one again)
    const int row = it.row0 + min(rt, nrows - 1);
    const int tok = row / a.G, hq = row - tok * a.G;
    const uint16_t* qp = a.q + (static_cast<int64_t>(it.q0) + tok) * a.q_t + (static_cast<int64_t>(head) * a.G + hq) * a.q_h + 8 * h;
    u32x4 qr[KM];
    float amax = 0.f;
#pragma unroll
    for (int m = 0; m < KM; ++m) {
        qr[m] = *reinterpret_cast<const u32x4*>(qp + 16 * m);
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(half_at<F16>(qr[m][i], 0)), fabsf(half_at<F16>(qr[m][i], 1))));
    }
    amax = xmax32(amax);
    if (!(amax < INFINITY)) amax = 0.f;
    const float most = xmax16(max16_dpp(amax)), least = -xmax16(max16_dpp(amax > 0.f ? -amax : -INFINITY));
    if (lane == 0) { L.red[0][w] = most; L.red[1][w] = least; }
    __syncthreads();
    float all_most = 0.f, all_least = INFINITY;
#pragma unroll
    for (int i = 0; i < CHUNK_WAVES; ++i) {
        all_most = fmaxf(all_most, L.red[0][i]);
        all_least = fminf(all_least, L.red[1][i]);
    }
    // One power of two for all rows.  Where some are below 2^-16 of the largest
    // (rare), they would lose bits of 2^-23 to it: then each row has its own, which the
    // careful path of `settle` applies to the scores (a product more per score in
    // the other path would cost 3%; so it is 1%, for the scores that live longer).
    const bool apart = __builtin_amdgcn_readfirstlane(all_least < all_most * 0x1p-16f);
    const int qe = q_exponent(apart ? amax : all_most);
    const float qs = pow2(-qe), row_scale = pow2(qe), qk = apart ? a.scale : a.scale * row_scale;
    f16x8 qop[KM];
#pragma unroll
    for (int m = 0; m < KM; ++m) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = half_at<F16>(qr[m][i >> 1], i & 1) * qs;
        qop[m] = f16x8{static_cast<_Float16>(f[0]), static_cast<_Float16>(f[4]), static_cast<_Float16>(f[1]), static_cast<_Float16>(f[5]),
                       static_cast<_Float16>(f[2]), static_cast<_Float16>(f[6]), static_cast<_Float16>(f[3]), static_cast<_Float16>(f[7])};
    }
    const int pos = it.len - it.qlen + tok;
    const int lo = first_key(pos, a.window), top = min(pos, it.key1 - 1);
    // every row of this wavefront sees [all_lo, all_hi]
    const int t0 = (it.row0 + min(32 * w, nrows - 1)) / a.G, t1 = (it.row0 + min(32 * w + 31, nrows - 1)) / a.G;
    const int all_hi = apart ? -1 : min(it.len - it.qlen + t0, it.key1 - 1), all_lo = first_key(it.len - it.qlen + t1, a.window);

    // ---- conversion ----
    // Wavefronts 0..3 have the V codes and scales of the 16-key tiles 0..3 of a
    // block, wavefronts 4..7 the K codes and scales: one page id and one
    // descriptor each, of range 0 (zeros, no access) where the page is not in
    // the pool.
    const bool is_v = w < 4;
    const int tile = w & 3;
    const int64_t hk = head * a.ps_head, hs = head * a.ss_head;
    const int page_mask = (1 << a.page_log2) - 1;
    const int32_t* trow = a.table + it.req * a.bt_stride;
    const int nblk = a.num_pages > 0 ? (max(it.key1 - it.key0, 0) + BLK - 1) / BLK : 0;
    // lane = key of the tile * KL + 32-channel part kq (D = 64: the upper 32
    // lanes store what the lower ones store)
    constexpr int KL = D / 32;
    const int cl = D == 128 ? lane : lane & 31;
    const int kkey = cl / KL, kq = cl % KL;
    const int8_t* const codes = is_v ? a.vp : a.kp;
    const uint16_t* const scales = is_v ? a.vs : a.ks;
    uint8_t* const mine = (is_v ? L.v[0] + (16 * tile + kkey) * VROW<D> : L.k[0] + (16 * tile + kkey) * KROW<D>) + 64 * kq;
    auto tile_key = [&](int blk) { return it.key0 + BLK * blk + 16 * tile; };
    auto page_id = [&](int blk) -> int { return trow[min(tile_key(blk), it.key1 - 1) >> a.page_log2]; };
    u32x4 raw = {};                      // 32 codes
    uint32_t sraw = 0;                   // scale bits (lanes 0..15)
    bool sok = false;                    // the page is in the pool
    auto fetch = [&](int blk, int id) __attribute__((always_inline)) {
        id = __builtin_amdgcn_readfirstlane(id);
        sok = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_pages);
        const int64_t pg = sok ? id : 0;
        const int o = (min(tile_key(blk), it.key1 - 1) & page_mask) & ~15;
        const Rsrc rc = make_rsrc(codes + pg * a.ps_page + hk + o * ROWB, sok ? 16 * ROWB : 0);
        const Rsrc rs = make_rsrc(scales + pg * a.ss_page + hs + o, sok ? 32 : 0);
        raw = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, 16 * cl, 0, 0));
        sraw = __builtin_amdgcn_raw_buffer_load_b16(rs, 2 * lane, 0, 0);
    };
    // block blk into buffer b
    auto store = [&](int blk, int b) __attribute__((always_inline)) {
        uint8_t* const dst = mine + b * (is_v ? sizeof(L.v[0]) : sizeof(L.k[0]));
        // a word's channels in the order 0, 4, 1, 5, 2, 6, 3, 7: the queries'
        // and, for V, that of the output's rows
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x4*>(dst + 16 * i) = u32x4{codes2(raw[i], 0), codes2(raw[i], 4), codes2(raw[i], 8), codes2(raw[i], 12)};
        const float f = f16_bits_to_f32(static_cast<uint16_t>(sraw));
        if (is_v) {
            // keys past the piece or in no page hold anything: they count as 0
            const bool live = lane < 16 && tile_key(blk) + lane < it.key1 && sok;
            const bool bad = live && !(fabsf(f) < INFINITY);
            const float x = live && !bad ? f : 0.f;
            const uint32_t mask = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(bad));
            const float e = scale_bound(fabsf(x)), most = max16_dpp(e), least = -max16_dpp(-e);
            if (lane < 16) L.vs[b][16 * tile + lane] = x;
            if (lane == 0) {
                L.ve[b][tile] = most + (mask || !sok || most - least > FAR ? BAD : 0.f);
                L.care[b][tile] = mask | (sok ? 1u << 16 : 0u);
            }
        } else if (lane < 16) {
            L.ks[b][16 * tile + lane] = f * qk;
        }
    };

    float m_run = M_INIT, l_run = 0.f;
    f32x16 acc[DT], sc;
    float t[16];                         // score - reference of 32 keys, then their weights
    uint32_t pw[8];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

    // K of half x, step m: key 32 x + (l & 31), channels 16 m + 8 h ..
    const uint8_t* const kl = L.k[0] + r32 * KROW<D> + 16 * h;
    // V of half x, step s, tile d: within 16 lanes, lane j of the transposing
    // read gets element j & 3 of the 8-byte pieces that the lanes 4 e + (j >> 2)
    // address: piece q = l & 3 of channels 32 d + (l & 16) + 4 q .. of key 32 x +
    // 16 s + 4 h + e (and 8 keys on), e = (l >> 2) & 3, which gives lane l
    // channel 32 d + (l & 31) of the keys of its registers 8 s ..
    const uint8_t* const vl = L.v[0] + (4 * h + ((lane >> 2) & 3)) * VROW<D> + 2 * (lane & 16) + 8 * (lane & 3);
    auto v_operand = [&](const uint8_t* p) __attribute__((always_inline)) {
        typedef short i16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) i16x4* LdsV;
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV)(p)));
        const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV)(p + 8 * VROW<D>)));
        return __builtin_bit_cast(f16x8, u32x4{x[0], x[1], y[0], y[1]});
    };
    auto qk_product = [&](int b, int x) __attribute__((always_inline)) {
        const uint8_t* const p = kl + b * static_cast<int>(sizeof(L.k[0]));
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
        for (int m = 0; m < KM; ++m)
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8*>(p + 32 * x * KROW<D> + 32 * m), qop[m], sc, 0, 0, 0);
    };
    auto pv_product = [&](int b, int x) __attribute__((always_inline)) {
        const uint8_t* const p = vl + b * static_cast<int>(sizeof(L.v[0]));
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const u32x4 pv = {pw[4 * s], pw[4 * s + 1], pw[4 * s + 2], pw[4 * s + 3]};
#pragma unroll
            for (int d = 0; d < DT; ++d)
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_operand(p + (32 * x + 16 * s) * VROW<D> + 64 * d), __builtin_bit_cast(f16x8, pv),
                                                                acc[d], 0, 0, 0);
        }
    };
    // t = scale * S - reference (0 while the row has seen no key); the lane's
    // largest + log2 of the largest V scale, 16-key tile by tile (t[0..7], t[8..15])
    auto scores = [&](int b, int x, float m_use) __attribute__((always_inline)) -> float {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 k4 = *reinterpret_cast<const f32x4*>(&L.ks[b][32 * x + 8 * g + 4 * h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) t[4 * g + i] = __builtin_fmaf(sc[4 * g + i], k4[i], -m_use);
        }
        float mx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float* u = t + 8 * i;
            mx[i] = vmax3(vmax3(u[0], u[1], u[2]), u[3], u[4]);
            mx[i] = vmax2(vmax3(mx[i], u[5], u[6]), u[7]) + L.ve[b][2 * x + i];
        }
        return vmax2(mx[0], mx[1]);
    };
    // hides what the rows do not see, and raises their reference where a
    // score passes it
    auto settle = [&](int b, int x, int blk, float mx, float m_use, bool unset) __attribute__((always_inline)) {
        const int j0 = it.key0 + BLK * blk + 32 * x;
        const float ve = fmaxf(L.ve[b][2 * x], L.ve[b][2 * x + 1]);
        if (j0 + 31 > all_hi || j0 < all_lo || __builtin_amdgcn_readfirstlane(__float_as_int(ve)) >= __float_as_int(BAD / 2)) {
            // the row's bound is over the V scales that it sees, so that what
            // is hidden from a row does not touch its bits; a row that sees a
            // scale that is not finite is NaN (its lse is not: l stays)
            bool nan = false;
            mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v4 = *reinterpret_cast<const f32x4*>(&L.vs[b][32 * x + 8 * g + 4 * h]);
                const uint32_t keys = L.care[b][2 * x + (g >> 1)];
                const uint32_t bad = keys >> (8 * (g & 1) + 4 * h);
                const bool in_pool = keys >> 16;
                if (apart) {             // (again, with the row's own power of two)
                    const f32x4 k4 = *reinterpret_cast<const f32x4*>(&L.ks[b][32 * x + 8 * g + 4 * h]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) t[4 * g + i] = __builtin_fmaf(sc[4 * g + i] * row_scale, k4[i], -m_use);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + 8 * g + 4 * h + i;
                    const bool seen = j <= top && j >= lo && in_pool;
                    t[4 * g + i] = seen ? t[4 * g + i] : -INFINITY;
                    mx = fmaxf(mx, t[4 * g + i] + scale_bound(fabsf(v4[i])));
                    nan |= seen && ((bad >> i) & 1);
                }
            }
            if (__builtin_amdgcn_ballot_w64(nan)) {
                const auto both = __builtin_amdgcn_permlane32_swap(nan, nan, false, false);      // (a row's two lanes)
                const float z = both[0] | both[1] ? __builtin_nanf("") : 0.f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d] += z;
            }
        }
        // (a row's own scores alone decide whether its reference moves)
        if (__builtin_amdgcn_ballot_w64(unset || mx > P_SHIFT + SLACK_W)) {      // rare after the first keys
            mx = xmax32(mx);
            const bool move = unset ? mx > -INFINITY : mx > P_SHIFT + SLACK_W;
            const float up = move ? mx - P_SHIFT : 0.f;
            const float alpha = unset ? 1.0f : fast_exp2(-up);
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= alpha;
            m_run = move ? m_use + up : m_run;
#pragma unroll
            for (int i = 0; i < 16; ++i) t[i] -= up;
        }
    };
    // P' = fp16(2^t * V scale) of half x (every scale in vs is finite: a hidden
    // key's weight of zero stays zero)
    auto weights = [&](int b, int x) __attribute__((always_inline)) {
        float ls[2] = {0.f, 0.f};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 v4 = *reinterpret_cast<const f32x4*>(&L.vs[b][32 * x + 8 * g + 4 * h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[4 * g + i] = fast_exp2(t[4 * g + i]);
                ls[i & 1] += t[4 * g + i];
            }
            pw[2 * g] = pack_f16x2(t[4 * g] * v4[0], t[4 * g + 1] * v4[1]);
            pw[2 * g + 1] = pack_f16x2(t[4 * g + 2] * v4[2], t[4 * g + 3] * v4[3]);
        }
        l_run += ls[0] + ls[1];
    };
    // One step: the next 32 keys' scores are multiplied while these 32 are
    // weighted, and formed while these are added up, so that the matrix and the
    // vector pipe have work at the same time.
    auto step = [&](int kb, int kx, int kblk, int vb, int vx) __attribute__((always_inline)) {
        qk_product(kb, kx);
        weights(vb, vx);
        const bool unset = m_run == M_INIT;
        const float m_use = unset ? 0.f : m_run;
        pv_product(vb, vx);
        const float mx = scores(kb, kx, m_use);
        settle(kb, kx, kblk, mx, m_use, unset);
    };

    if (nblk > 0) {
        fetch(0, page_id(0));
        store(0, 0);
        fetch(1, page_id(1));
        store(1, 1);
        fetch(2, page_id(2));
        int id = page_id(3);
        __syncthreads();
        qk_product(0, 0);
        settle(0, 0, 0, scores(0, 0, 0.f), 0.f, true);
        // one wavefront of a SIMD goes first where both could issue: they drift
        // half a step apart
        if (w < CHUNK_WAVES / 2) __builtin_amdgcn_s_setprio(1);
        int b0 = 0, b1 = 1, b2 = 2;      // buffers of the blocks n, n + 1, n + 2
        for (int n = 0; n < nblk; ++n) {
            store(n + 2, b2);
            fetch(n + 3, id);
            id = page_id(n + 4);
            step(b0, 1, n, b0, 0);
            step(b1, 0, n + 1, b0, 1);   // (past the last block: hidden keys)
            const int o = b0;
            b0 = b1;
            b1 = b2;
            b2 = o;
            __syncthreads();
        }
    }
    if (rt >= nrows) return;
    const auto lr = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
    l_run = __uint_as_float(lr[0]) + __uint_as_float(lr[1]);
    // Registers 4 g .. of a tile are the rows 8 g + 4 h ..: channels 0, 4, 1, 5 (h =
    // 0) or 2, 6, 3, 7 of 8: two values change places between the lane's halves
    const int64_t at = (static_cast<int64_t>(it.part) * a.heads + head) * CHUNK + rt;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 o = {acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
            const float x = __shfl_xor(h ? o[0] : o[1], 32, 64), y = __shfl_xor(h ? o[2] : o[3], 32, 64);
            const f32x4 z = h ? f32x4{x, y, o[1], o[3]} : f32x4{o[0], o[2], x, y};
            const int ch = 32 * d + 8 * g + 4 * h;
            if (it.part >= 0) *reinterpret_cast<f32x4*>(a.part + at * D + ch) = z;
            else store_row<F16>(a, it.q0, row, head, ch, m_run, l_run, z);
        }
    if (it.part >= 0 && h == 0) { a.ml[at * 2] = m_run; a.ml[at * 2 + 1] = l_run; }
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

int check_pool(const char* what, int32_t head_dim, int32_t page_size, int64_t num_pages, int32_t kv_heads, const void* kp,
               const void* vp, const void* ks, const void* vs, int64_t ps_page, int64_t ps_head, int64_t ss_page,
               int64_t ss_head) {
    const std::string w = std::string(what) + ": ";
    if (head_dim != 64 && head_dim != 128) return fail(HYQ_ENOTSUP, w + "head_dim must be 64 or 128, got " + std::to_string(head_dim));
    if (!ok_page(page_size)) return fail(HYQ_ENOTSUP, w + "page_size must be a power of two from 16 to 256, got " + std::to_string(page_size));
    if (num_pages < 0 || num_pages > (int64_t{1} << 30)) return fail(HYQ_EINVAL, w + "num_pages out of range");
    if (kv_heads < 1 || kv_heads > 65535) return fail(HYQ_EINVAL, w + "key heads out of range");
    if (num_pages == 0) return HYQ_OK;
    if (!kp || !vp || !ks || !vs) return fail(HYQ_EINVAL, w + "null cache pointer");
    if (!aligned(kp, 16) || !aligned(vp, 16) || ps_page % 16 || ps_head % 16)
        return fail(HYQ_EINVAL, w + "code pages must be 16-byte aligned with strides divisible by 16");
    if (!aligned(ks, 2) || !aligned(vs, 2)) return fail(HYQ_EINVAL, w + "scales misaligned");
    return HYQ_OK;
}

// a launch has fewer than 2^32 threads along a dimension
constexpr int64_t MOST_THREADS = (int64_t{1} << 32) - 1024;
int64_t most_rows(int head_dim) { return MOST_THREADS / (head_dim / 8); }

int check_attention(const hyq_paged_params* p) {
    const char* w = "hyq_paged_attention";
    if (!p) return fail(HYQ_EINVAL, std::string(w) + ": null parameters");
    const std::string s = std::string(w) + ": ";
    if (int st = check_pool(w, p->head_dim, p->page_size, p->num_pages, p->kv_heads, p->k_pages, p->v_pages, p->k_scale, p->v_scale,
                            p->p_stride_page, p->p_stride_head, p->s_stride_page, p->s_stride_head))
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

template <int D, bool F16>
int launch_attention(AttnArgs a, const PlanArgs& narrow, const PlanArgs& wide, const Both& s, char* ws, hipStream_t st) {
    auto partials = [&](const Sizes& z) {
        a.part = reinterpret_cast<float*>(ws + z.off_part);
        a.ml = reinterpret_cast<float*>(ws + z.off_ml);
    };
    if (s.wide.items) {
        a.plan = wide;
        partials(s.wide);
        static std::atomic<uint64_t> raised{0};
        if (int rc = raise_lds(reinterpret_cast<const void*>(paged_chunk_kernel<D, F16>), sizeof(ChunkLds<D>), raised)) return rc;
        paged_chunk_kernel<D, F16><<<dim3(static_cast<unsigned>(s.wide.items * a.heads)), dim3(64 * CHUNK_WAVES), sizeof(ChunkLds<D>), st>>>(a);
    }
    a.plan = narrow;
    partials(s.narrow);
    if (s.narrow.items) paged_attn_kernel<D, F16><<<dim3(static_cast<unsigned>(s.narrow.items), a.heads), dim3(64 * WAVES), 0, st>>>(a);
    // a round of resident workgroups (two a CU) for the kind that there is, half
    // of one each where both may be
    const int64_t most = s.narrow.joins && s.wide.joins ? 256 : 512;
    int64_t jn = a.counters ? 0 : join_grid<Narrow, D>(s.narrow, a.heads, most);
    const int64_t jw = join_grid<Wide, D>(s.wide, a.heads, most);
    if (a.zero_tail && a.plan.cu && jn + jw == 0) jn = 1;
    if (jn + jw)
        paged_join_kernel<D, F16><<<dim3(static_cast<unsigned>(jn + jw)), dim3(JOIN_T), 0, st>>>(
            a, wide, reinterpret_cast<float*>(ws + s.wide.off_part), reinterpret_cast<float*>(ws + s.wide.off_ml), static_cast<int>(jn));
    return check_launch("hyq_paged_attention");
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

}  // namespace
}  // namespace hyq

using namespace hyq;

extern "C" int hyq_paged_batch(const int32_t* context_lens, const int32_t* new_lens, int32_t num_requests,
                               int32_t* block_table, int64_t bt_stride, int32_t max_pages, const int32_t* free_pages,
                               int32_t num_free, int32_t page_size, int32_t num_tokens, int32_t* cu_seqlens,
                               int32_t* seq_lens, int64_t* slots, int64_t* positions, int32_t* pages_used, void* stream) {
    if (num_requests < 0 || num_tokens < 0 || max_pages < 0 || num_free < 0) return fail(HYQ_EINVAL, "hyq_paged_batch: negative size");
    if (num_requests > MAX_REQUESTS)
        return fail(HYQ_ENOTSUP, "hyq_paged_batch: at most " + std::to_string(MAX_REQUESTS) + " requests, got " + std::to_string(num_requests));
    if (!ok_page(page_size))
        return fail(HYQ_ENOTSUP, "hyq_paged_batch: page_size must be a power of two from 16 to 256, got " + std::to_string(page_size));
    if (!cu_seqlens || !pages_used || (num_requests && (!context_lens || !new_lens || !seq_lens)) ||
        (num_requests && max_pages && !block_table) || (num_free && !free_pages) || (num_tokens && (!slots || !positions)))
        return fail(HYQ_EINVAL, "hyq_paged_batch: null pointer");
    if (!aligned(context_lens, 4) || !aligned(new_lens, 4) || !aligned(block_table, 4) || !aligned(free_pages, 4) ||
        !aligned(cu_seqlens, 4) || !aligned(seq_lens, 4) || !aligned(pages_used, 4) || !aligned(slots, 8) || !aligned(positions, 8))
        return fail(HYQ_EINVAL, "hyq_paged_batch: misaligned pointer");
    // (a request's new entries would be written over another's)
    if (num_requests > 1 && bt_stride < max_pages && bt_stride > -static_cast<int64_t>(max_pages))
        return fail(HYQ_EINVAL, "hyq_paged_batch: rows of block_table share memory");
    BatchArgs a{context_lens, new_lens, block_table, bt_stride, free_pages, cu_seqlens, seq_lens, pages_used, slots, positions,
                num_requests, max_pages, num_free, log2i(page_size), num_tokens};
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(512, 1 + (static_cast<int64_t>(num_tokens) - 1) / BATCH_TOKENS));
    const size_t lds = 2 * (static_cast<size_t>(num_requests) + 1) * sizeof(int32_t);
    static std::atomic<uint64_t> raised{0};
    if (lds > 64 * 1024 - 64)
        if (int rc = raise_lds(reinterpret_cast<const void*>(paged_batch_kernel), 2 * (MAX_REQUESTS + 1) * sizeof(int32_t), raised)) return rc;
    paged_batch_kernel<<<dim3(blocks), dim3(BT), lds, static_cast<hipStream_t>(stream)>>>(a);
    return check_launch("hyq_paged_batch");
}

extern "C" int hyq_paged_append(const uint16_t* k, int64_t k_stride_t, int64_t k_stride_h, const uint16_t* v, int64_t v_stride_t,
                                int64_t v_stride_h, int32_t is_fp16, const int64_t* slots, int64_t num_tokens, int32_t kv_heads,
                                int32_t head_dim, int8_t* k_pages, int8_t* v_pages, int64_t p_stride_page, int64_t p_stride_head,
                                uint16_t* k_scale, uint16_t* v_scale, int64_t s_stride_page, int64_t s_stride_head,
                                int64_t num_pages, int32_t page_size, void* stream) {
    if (int st = check_pool("hyq_paged_append", head_dim, page_size, num_pages, kv_heads, k_pages, v_pages, k_scale, v_scale, p_stride_page,
                            p_stride_head, s_stride_page, s_stride_head))
        return st;
    if (num_tokens < 0) return fail(HYQ_EINVAL, "hyq_paged_append: negative size");
    if (is_fp16 != 0 && is_fp16 != 1) return fail(HYQ_EINVAL, "hyq_paged_append: is_fp16 must be 0 or 1");
    if (num_tokens == 0 || num_pages == 0) return HYQ_OK;
    if (!k || !v || !slots) return fail(HYQ_EINVAL, "hyq_paged_append: null pointer");
    if (!aligned(k, 16) || !aligned(v, 16) || (k_stride_t | k_stride_h | v_stride_t | v_stride_h) % 8 || !aligned(slots, 8))
        return fail(HYQ_EINVAL, "hyq_paged_append: rows must be 16-byte aligned with strides divisible by 8");
    if (num_tokens > most_rows(head_dim) / kv_heads)
        return fail(HYQ_ENOTSUP, "hyq_paged_append: more than " + std::to_string(most_rows(head_dim)) + " rows");
    const int64_t rows = num_tokens * kv_heads;
    RowArgs a{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, nullptr, nullptr, slots, k_pages, v_pages, p_stride_page, p_stride_head,
              k_scale, v_scale, s_stride_page, s_stride_head, num_pages * page_size, static_cast<uint32_t>(rows),
              static_cast<uint32_t>(kv_heads), log2i(page_size), log2i(head_dim / 8)};
    const int64_t per = 256 >> a.lpt_log2;
    const dim3 grid(static_cast<unsigned>((rows + per - 1) / per), 2);
    if (is_fp16) paged_append_kernel<true><<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a);
    else paged_append_kernel<false><<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a);
    return check_launch("hyq_paged_append");
}

extern "C" int hyq_paged_gather(const int64_t* slots, int64_t num_tokens, int32_t kv_heads, int32_t head_dim, const int8_t* k_pages,
                                const int8_t* v_pages, int64_t p_stride_page, int64_t p_stride_head, const uint16_t* k_scale,
                                const uint16_t* v_scale, int64_t s_stride_page, int64_t s_stride_head, int64_t num_pages,
                                int32_t page_size, int32_t out_fp16, uint16_t* k_out, uint16_t* v_out, void* stream) {
    if (int st = check_pool("hyq_paged_gather", head_dim, page_size, num_pages, kv_heads, k_pages, v_pages, k_scale, v_scale, p_stride_page,
                            p_stride_head, s_stride_page, s_stride_head))
        return st;
    if (num_tokens < 0) return fail(HYQ_EINVAL, "hyq_paged_gather: negative size");
    if (out_fp16 != 0 && out_fp16 != 1) return fail(HYQ_EINVAL, "hyq_paged_gather: out_fp16 must be 0 or 1");
    if (num_tokens == 0) return HYQ_OK;
    if (!k_out || !v_out || !slots) return fail(HYQ_EINVAL, "hyq_paged_gather: null pointer");
    if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(slots, 8)) return fail(HYQ_EINVAL, "hyq_paged_gather: misaligned pointer");
    if (num_tokens > most_rows(head_dim) / kv_heads)
        return fail(HYQ_ENOTSUP, "hyq_paged_gather: more than " + std::to_string(most_rows(head_dim)) + " rows");
    const int64_t rows = num_tokens * kv_heads;
    RowArgs a{nullptr, nullptr, 0, 0, 0, 0, k_out, v_out, slots, const_cast<int8_t*>(k_pages), const_cast<int8_t*>(v_pages), p_stride_page,
              p_stride_head, const_cast<uint16_t*>(k_scale), const_cast<uint16_t*>(v_scale), s_stride_page, s_stride_head,
              num_pages * page_size, static_cast<uint32_t>(rows), static_cast<uint32_t>(kv_heads), log2i(page_size), log2i(head_dim / 8)};
    const int64_t per = 256 >> a.lpt_log2;
    const dim3 grid(static_cast<unsigned>((rows + per - 1) / per), 2);
    if (out_fp16) paged_gather_kernel<true><<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a);
    else paged_gather_kernel<false><<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a);
    return check_launch("hyq_paged_gather");
}

extern "C" size_t hyq_paged_attention_workspace_size(const hyq_paged_params* p) {
    if (check_attention(p) != HYQ_OK || p->num_requests == 0 || p->num_tokens == 0) return 0;
    return sizes_of(*p).wide.end;
}

extern "C" int hyq_paged_attention(const hyq_paged_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = check_attention(p)) return st;
    if (p->num_requests == 0 || p->num_tokens == 0) return HYQ_OK;
    const Both s = sizes_of(*p);
    if (!workspace || workspace_bytes < s.wide.end)
        return fail(HYQ_ENOSPC, "hyq_paged_attention: workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(s.wide.end) + " needed");
    if (!aligned(workspace, 256)) return fail(HYQ_EINVAL, "hyq_paged_attention: workspace must be 256-byte aligned");
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
    // calls with counters are numbered in the order of their launches
    static std::mutex order;
    static uint64_t calls = 0;
    const bool here = join_here(*p, s, st);
    std::unique_lock<std::mutex> lock(order, std::defer_lock);
    if (here) lock.lock();
    const uint64_t call = here ? ++calls : 0;
    const AttnArgs a{static_cast<const uint16_t*>(p->q), p->q_stride_t, p->q_stride_h, static_cast<uint16_t*>(p->out), p->o_stride_t, p->o_stride_h,
                     p->lse, static_cast<int64_t>(p->kv_heads) * p->kv_repeat, p->k_pages, p->v_pages, p->p_stride_page, p->p_stride_head,
                     p->k_scale, p->v_scale, p->s_stride_page, p->s_stride_head, p->block_table, p->bt_stride, narrow, nullptr, nullptr,
                     here ? reinterpret_cast<uint64_t*>(p->counters) : nullptr, call << CALL_SHIFT, p->kv_repeat, p->kv_heads, log2i(p->page_size), static_cast<int32_t>(p->num_pages), window, p->zero_tail,
                     p->sm_scale * 1.44269504f};
    if (p->head_dim == 128) return p->dtype_fp16 ? launch_attention<128, true>(a, narrow, wide, s, ws, st) : launch_attention<128, false>(a, narrow, wide, s, ws, st);
    return p->dtype_fp16 ? launch_attention<64, true>(a, narrow, wide, s, ws, st) : launch_attention<64, false>(a, narrow, wide, s, ws, st);
}
