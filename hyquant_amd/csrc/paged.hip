// The paged 4-bit KV cache: batch layout, append, read-back and attention
// over block tables.
//
// Cache: int8 [pages, key heads, page, D/2] codes of hyq_quant_pack's 4-bit
// format (the even channel in the low nibble) and fp16 [pages, key heads,
// page] scales, K and V alike; token j of request r sits in page
// block_table[r][j / page] at row j % page.  Pages are a power of two of 16
// to 256 tokens, so a 16-token tile never crosses a page and every tile's
// rows are one base address plus 32-bit lane offsets; bases are 64-bit.
#include "paged_attn.h"

namespace hyq {

CallOrder& call_order() {
    static CallOrder order;
    return order;
}

namespace {

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
constexpr int MAX_REQUESTS = 16384;      // two int32 prefix arrays of a batch fit in LDS
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

// ---------------------------------------------------------------------------
// attention: 16 query rows per workgroup
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t nib2(uint32_t x, int s, uint32_t magic) { return ((x >> s) & 0x000f000fu) ^ magic; }
template <int I>
__device__ __forceinline__ float quad_bcast(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), I * 0x55, 0xf, 0xf, true));
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
    const uint16_t *const ks = static_cast<const uint16_t*>(a.ks), *const vs = static_cast<const uint16_t*>(a.vs);
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
            const Rsrc rks = make_rsrc(ks + so, in ? 32 : 0), rvs = make_rsrc(vs + so, in ? 32 : 0);
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
    finish_tile<D, F16>(a, it, head, nrows, red, redm, redl);
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
constexpr float BAD = 4096.0f;
constexpr float FAR = 8.0f;              // binary orders that the V scales of 16 keys may span

__device__ __forceinline__ uint32_t pk_sub1032(uint32_t x) {
    const f16x2 b = {static_cast<_Float16>(1032.0f), static_cast<_Float16>(1032.0f)};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - b);
}
// two codes of a word as fp16: 1024 + (nibble ^ 8) is exact, so is minus 1032
__device__ __forceinline__ uint32_t codes2(uint32_t x, int s) { return pk_sub1032(nib2(x, s, 0x64086408u)); }
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
    const uint16_t* const scales = static_cast<const uint16_t*>(is_v ? a.vs : a.ks);
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

template <int D, bool F16>
struct Kernels {
    static auto narrow(const AttnArgs&) { return paged_attn_kernel<D, F16>; }
    static constexpr auto chunk = paged_chunk_kernel<D, F16>;
    static constexpr size_t chunk_lds = sizeof(ChunkLds<D>);
};

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
    if (int st = check_pool("hyq_paged_append", 2, head_dim, page_size, num_pages, kv_heads, k_pages, v_pages, k_scale, v_scale, p_stride_page,
                            p_stride_head))
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
    if (int st = check_pool("hyq_paged_gather", 2, head_dim, page_size, num_pages, kv_heads, k_pages, v_pages, k_scale, v_scale, p_stride_page,
                            p_stride_head))
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
    return attention_workspace("hyq_paged_attention", 2, p);
}

extern "C" int hyq_paged_attention(const hyq_paged_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    return attention<Kernels>("hyq_paged_attention", 2, p, workspace, workspace_bytes, stream);
}
