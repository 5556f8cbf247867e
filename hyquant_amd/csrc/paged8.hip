// Attention over the paged 8-bit KV cache.
//
// Cache: int8 [pages, key heads, page, D] codes and fp32 [pages, key heads, page /
// 16] scales, K and V alike: a scale for each block of 16 tokens and head, which
// is a tile of the kernels.  Pages, tables and the schedule are those of the 4-bit
// cache.
#include "paged_attn.h"

namespace hyq {
namespace {

constexpr uint32_t FLIP = 0x80808080u;   // signed codes to u = code + 128
constexpr float SCALE_MIN = 0x1p-40f, SCALE_MAX = 0x1p48f;
constexpr float P_TOP = 6.0f;            // a row's reference is its largest score + log2 V scale, less this

// A scale outside of these bounds makes whatever sees it NaN; a hidden key's
// weight is selected.
__device__ __forceinline__ float checked(float s) { return __builtin_amdgcn_fmed3f(s, SCALE_MIN, SCALE_MAX) == s ? s : __builtin_nanf(""); }
// bytes b and b + 1 of x, or byte b of x and of y, as the fp16 subnormals u 2^-24
template <int B> __device__ __forceinline__ uint32_t bytes2(uint32_t x) {
    return __builtin_amdgcn_perm(0u, x, 0x0c000c00u | (B + 1) << 16 | B);
}
template <int B> __device__ __forceinline__ uint32_t bytes2(uint32_t x, uint32_t y) {
    return __builtin_amdgcn_perm(y, x, 0x0c000c00u | (B + 4) << 16 | B);
}
__device__ __forceinline__ uint32_t pack_rtz(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
__device__ __forceinline__ float f16_at(uint32_t w, int hi) { return f16_bits_to_f32(static_cast<uint16_t>(hi ? w >> 16 : w)); }

// ---------------------------------------------------------------------------
// 16 query rows per workgroup
// ---------------------------------------------------------------------------
// A workgroup has one KV head of a tile of 16 rows (a request's tokens times the
// G query heads) and a range of keys; its four wavefronts take every fourth
// 32-key step and join through LDS at the end.
//   QK  S^T[key][row] = K . Q^T with v_mfma_f32_16x16x32_f16.  A K operand is
//       u = code + 128 as the fp16 subnormal u 2^-24, a byte permute per pair of
//       codes; the accumulators start at -128 sum(q) 2^-24.
//   softmax: t = score + log2(V scale) - M, P' = 2^t = p v_scale 2^-M: a tile's
//       scales are one number each, so that they cost one fma.  M follows the
//       row's own largest t, and l sums P' / v_scale.
//   PV  O^T[channel][row] = V^T . P'^T with the same instruction, V operands
//       u 2^-24 again, P' as the sum of two fp16 numbers (2^-21 of a weight is
//       lost; one fp16 number would be 2^-12 of it, as much as an fp16 output's own
//       rounding); 128 sum(P') is taken off every RING steps of a wavefront, by
//       products with a constant, before its fp32 roundings add up.
// Bound by the cache's bytes: 16 requests of 32K keys (1.08 GB) take 172 to 174 us, 6.2
// TB/s, where a copy reaches 5.05 and a stream of reads alone 6.8.  48 requests of 700 to
// 32000 keys in pages of 16 149 us (5.15 TB/s; in pages of 64 146): pieces of unequal
// length.  Short calls are bound by the chain lengths -> table -> rows -> pieces: 12.7
// us for one request of 8K keys.
template <int D>
struct Raw8 {
    uint32_t k[2][D / 16];               // tile t: channels 16 kb .. and 64 + 16 kb .. of token 16t + 4(c & 3) + (c >> 2)
    uint32_t v[8][D / 64];               // slot e: token 4e + kb, channels (D/16) c ..
    uint32_t sk[2], sv[2];               // tile t: scale bits
    int first;                           // first token of the group
    int ok;                              // bit t: tile t's page is inside the pool
};
constexpr int RING = 2;                  // groups in registers (three leave room for 2 workgroups a CU instead of 3: 13.2 us instead of 12.7 for one request of 8K, 37 instead of 31 for 200 of heads of 64)

// PAIR: pages hold a whole group of 32 keys, so that a group has one page id and one
// address instead of two.
template <int D, bool F16, bool PAIR>
__global__ __launch_bounds__(64 * WAVES, D == 64 ? 4 : 3) void paged8_attn_kernel(AttnArgs a) {
    constexpr int TILE = Narrow::TILE, GROUP = Narrow::GROUP;
    constexpr int NB = D / 16;           // PV products per group
    constexpr int KM = D / 32;           // QK products per tile
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
    const uint16_t* qp = a.q + (static_cast<int64_t>(it.q0) + tok) * a.q_t + (static_cast<int64_t>(head) * a.G + hq) * a.q_h + 16 * kb;
    const int32_t* trow = a.table + it.req * a.bt_stride;
    const int steps = (max(it.key1 - it.key0, 0) + GROUP - 1) / GROUP;
    const int mine = steps > w && a.num_pages > 0 ? (steps - w + WAVES - 1) / WAVES : 0;   // this wavefront's groups w, w + 4, ...
    // page ids of this wavefront's next SPAN groups: of group i in lane i, or of its tile t in lane 2i + t
    constexpr int IDS = PAIR ? 1 : 2, SPAN = 64 / IDS;
    auto ids_at = [&](int i0) -> int {
        const int t = it.key0 + GROUP * (w + WAVES * (i0 + lane / IDS)) + 16 * (lane & (IDS - 1));
        return trow[min(t, it.key1 - 1) >> a.page_log2];
    };
    int ids = 0, ids_next = 0;
    if (mine > 0) ids = ids_at(0);
    if (mine > SPAN) ids_next = ids_at(SPAN);
    u32x4 qr[KM];
#pragma unroll
    for (int m = 0; m < KM; ++m) qr[m] = *reinterpret_cast<const u32x4*>(qp + 64 * (m >> 1) + 8 * (m & 1));

    const int64_t hk = head * a.ps_head, hs = head * a.ss_head;
    const float *const ks = static_cast<const float*>(a.ks), *const vs = static_cast<const float*>(a.vs);
    const int page_mask = (1 << a.page_log2) - 1;
    const uint32_t klane = (4 * (c & 3) + (c >> 2)) * D + 16 * kb;
    const uint32_t vlane = kb * D + (D / 16) * c;
    // Every load goes through a buffer descriptor over its 16-token tile, of
    // range 0 past this wavefront's groups or where the page is not in the
    // pool: such loads give zeros and touch no memory.
    auto load = [&](Raw8<D>& r, int i) {
        if (i > 0 && (i & (SPAN - 1)) == 0) {
            ids = ids_next;
            ids_next = mine > i + SPAN ? ids_at(i + SPAN) : 0;
        }
        r.first = it.key0 + GROUP * (w + WAVES * i);
        r.ok = 0;
#pragma unroll
        for (int u = 0; u < IDS; ++u) {
            constexpr int TILES = 2 / IDS;
            const int id = __builtin_amdgcn_readlane(ids, IDS * (i & (SPAN - 1)) + u);
            const bool ok = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_pages);
            const bool in = ok && i < mine;
            r.ok |= ok ? (PAIR ? 3 : 1 << u) : 0;
            const int64_t pg = ok ? id : 0;
            const int t0 = (min(r.first + 16 * u, it.key1 - 1) & page_mask) & ~(16 * TILES - 1);
            const int64_t co = pg * a.ps_page + hk + t0 * D, so = pg * a.ss_page + hs + (t0 >> 4);
            const Rsrc rk = make_rsrc(a.kp + co, in ? 16 * TILES * D : 0), rv = make_rsrc(a.vp + co, in ? 16 * TILES * D : 0);
            const Rsrc rks = make_rsrc(ks + so, in ? 4 * TILES : 0), rvs = make_rsrc(vs + so, in ? 4 * TILES : 0);
#pragma unroll
            for (int x = 0; x < TILES; ++x) {
                const int t = PAIR ? x : u;
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, klane + 64 * j + 16 * D * x, 0, NT));
                    r.k[t][4 * j] = v[0]; r.k[t][4 * j + 1] = v[1]; r.k[t][4 * j + 2] = v[2]; r.k[t][4 * j + 3] = v[3];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (D == 128) {
                        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, vlane + (4 * e + 16 * x) * D, 0, NT));
                        r.v[4 * t + e][0] = v[0];
                        r.v[4 * t + e][1] = v[1];
                    } else {
                        r.v[4 * t + e][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, vlane + (4 * e + 16 * x) * D, 0, NT);
                    }
                }
            }
            if constexpr (PAIR) {
                const u32x2 k2 = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rks, 0, 0, 0));
                const u32x2 v2 = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rvs, 0, 0, 0));
                r.sk[0] = k2[0]; r.sk[1] = k2[1];
                r.sv[0] = v2[0]; r.sv[1] = v2[1];
            } else {
                r.sk[u] = __builtin_amdgcn_raw_buffer_load_b32(rks, 0, 0, 0);
                r.sv[u] = __builtin_amdgcn_raw_buffer_load_b32(rvs, 0, 0, 0);
            }
        }
    };
    Raw8<D> ring[RING];
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) load(ring[i], i);

    // ---- queries: B operands, row c's channels 64 (m >> 1) + 16 kb + 8 (m & 1) .. ----
    float amax = 0.f;
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(half_at<F16>(qr[m][i], 0)), fabsf(half_at<F16>(qr[m][i], 1))));
    // (a power of two of each row's own: rows of any magnitude stand side by side)
    amax = col_max(amax);
    if (!(amax < INFINITY)) amax = 0.f;
    const int qe = q_exponent(amax);
    const float qs = pow2(-qe), row_scale = pow2(qe);
    f16x8 qop[KM];
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) qop[m][i] = static_cast<_Float16>(half_at<F16>(qr[m][i >> 1], i & 1) * qs);
    const float qk = a.scale * 16777216.0f;                // K operands are u * 2^-24
    f32x4 kbias = {0.f, 0.f, 0.f, 0.f};
    const u32x4 offset = {0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u};     // 128 * 2^-24
#pragma unroll
    for (int m = 0; m < KM; ++m) kbias = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, offset), qop[m], kbias, 0, 0, 0);
    kbias = -kbias;
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

    auto compute = [&](const Raw8<D>& r) {
        float s[8], sk[2], lv[2], vinv[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            sk[t] = checked(__uint_as_float(r.sk[t])) * qk * row_scale;
            const float v = checked(__uint_as_float(r.sv[t]));
            lv[t] = __builtin_amdgcn_logf(v);
            vinv[t] = __builtin_amdgcn_rcpf(v);
            f32x4 x = kbias;
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                const uint32_t k0 = r.k[t][2 * m] ^ FLIP, k1 = r.k[t][2 * m + 1] ^ FLIP;
                const u32x4 o = {bytes2<0>(k0), bytes2<2>(k0), bytes2<0>(k1), bytes2<2>(k1)};
                x = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, o), qop[m], x, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * t + i] = __builtin_fmaf(x[i], sk[t], lv[t]);
        }
        // masked keys: behind the row's own position or before its window,
        // past the piece, or in a page outside the pool.  Their scores and
        // weights are selected: what is there may be anything.
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
        mx = vmax2(mx, s[7]) - P_TOP;
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
        for (int e = 0; e < 8; ++e) s[e] = fast_exp2(s[e] - m_run);
        if (edge) {
#pragma unroll
            for (int t = 0; t < 2; ++t) vinv[t] = ((dead >> (4 * t)) & 15) == 15 ? 0.f : vinv[t];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = (dead >> e) & 1 ? 0.f : s[e];
        }
        l_run = __builtin_fmaf((s[0] + s[1]) + (s[2] + s[3]), vinv[0], l_run);
        l_run = __builtin_fmaf((s[4] + s[5]) + (s[6] + s[7]), vinv[1], l_run);
        u32x4 ph, pl;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ph[i] = pack_rtz(s[2 * i], s[2 * i + 1]);
            pl[i] = pack_rtz(s[2 * i] - f16_at(ph[i], 0), s[2 * i + 1] - f16_at(ph[i], 1));
        }
        const f16x8 phi = __builtin_bit_cast(f16x8, ph), plo = __builtin_bit_cast(f16x8, pl);
        auto product = [&](f32x4& x, const u32x4& o) {
            x = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, o), phi, x, 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, o), plo, x, 0, 0, 0);
        };
#pragma unroll
        for (int d = 0; d < D / 64; ++d) {
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = r.v[e][d] ^ FLIP;
            product(acc[4 * d + 0], u32x4{bytes2<0>(v[0], v[1]), bytes2<0>(v[2], v[3]), bytes2<0>(v[4], v[5]), bytes2<0>(v[6], v[7])});
            product(acc[4 * d + 1], u32x4{bytes2<1>(v[0], v[1]), bytes2<1>(v[2], v[3]), bytes2<1>(v[4], v[5]), bytes2<1>(v[6], v[7])});
            product(acc[4 * d + 2], u32x4{bytes2<2>(v[0], v[1]), bytes2<2>(v[2], v[3]), bytes2<2>(v[4], v[5]), bytes2<2>(v[6], v[7])});
            product(acc[4 * d + 3], u32x4{bytes2<3>(v[0], v[1]), bytes2<3>(v[2], v[3]), bytes2<3>(v[4], v[5]), bytes2<3>(v[6], v[7])});
        }
        product(ones, offset);
    };
    for (int i = 0; i < mine; i += RING) {
#pragma unroll
        for (int j = 0; j < RING; ++j) {
            load(ring[(j + RING - 1) % RING], i + j + RING - 1);
            if (j == 0 || i + j < mine) compute(ring[j]);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[nb] -= ones;       // the codes' offset
        ones = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- the four wavefronts' results, joined through LDS ----
    l_run = col_sum(l_run);
    if (kb == 0) { redm[w][c] = m_run; redl[w][c] = l_run; }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[w][c][(D / 16) * (4 * kb + i) + nb] = acc[nb][i] * 16777216.0f;
    finish_tile<D, F16>(a, it, head, nrows, red, redm, redl);
}

// ---------------------------------------------------------------------------
// CHUNK query rows per workgroup
// ---------------------------------------------------------------------------
// A wavefront owns 32 rows.  The codes of 64 keys at a time are turned into
// fp16 operands once for all rows of the workgroup and laid in LDS, two blocks
// ahead of the products.
//   QK  S^T[key][row] = K . Q^T  with v_mfma_f32_32x32x16_f16, K operands u 2^-24
//       as above, queries (each row's scaled by a power of two of its own) exact.
//   t = (S - 128 2^-24 sum(q)) k_scale + log2(V scale) - M: a tile's scales, times
//       the row's power of two, and the offset are one fma's constants.
//   PV  O^T[channel][row] = V^T . P'^T, P' = fp16(2^t) against the exact codes,
//       V^T by transposing LDS reads.  M follows the row's own largest t, so that
//       P' keeps to [0, 2^13]; rounding P' to 11 bits once is the only rounding
//       between the scores and the output.  l sums 2^t / v_scale.  Against 64 bits
//       and relative to the outputs, bf16 is off by 1.67e-3 (its own rounding
//       1.66e-3), fp16 by 2.8e-4 (2.1e-4).  P' in two fp16 numbers, as above, leaves
//       the outputs' own roundings and takes 453 us where this takes 344 (2048 tokens
//       at 8192), 117 where this takes 98.6 (chunks beside decode steps).
// Bound by the matrix pipe, the LDS reads that feed it and the VALU work beside it:
// 2048 tokens at 8192 (309 GFLOP) take 334 to 362 us by box, 0.85 to 0.92 PFLOP/s where
// a large matrix product reaches 1.33; of 347 us on another box the products with their
// LDS reads alone took 224, with the conversion 267, with the softmax 311.  Both halves
// of a block are pipelined against each other, and the first four wavefronts have
// priority, as in the 4-bit kernel.
// Four wavefronts of 64 rows, one a SIMD, read LDS half as often but leave the pipes
// to one instruction stream: 542 us.  K and V converted by different wavefronts, K's
// offset taken off there: 342.
// Output register i of a lane (row l & 31, half h = l >> 5) of a 32-key product
// is key 8 (i >> 2) + 4 h + (i & 3); registers 8s .. 8s + 7 are the B operand of
// step s of P.V, without a shuffle.
template <int D>
struct ChunkLds8 {
    uint8_t k[BUFS][BLK * KROW<D>];
    uint8_t v[BUFS][BLK * VROW<D>];
    float ks[BUFS][4];                   // per 16-key tile: K scale * scale * 2^24, or NaN
    float lv[BUFS][4], vi[BUFS][4];      // log2 of the V scale, or NaN; its inverse, or 0
    uint32_t in[BUFS][4];                // the page is in the pool
};

// bytes b and b + 1 of u = code + 128 as fp16 codes (V's): 1024 + u is exact, so is minus 1152
template <int B> __device__ __forceinline__ uint32_t codes2(uint32_t u) {
    const f16x2 x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04000400u | (B + 1) << 16 | B));
    const f16x2 b = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    return __builtin_bit_cast(uint32_t, x - b);
}

template <int D, bool F16>
__global__ __launch_bounds__(64 * CHUNK_WAVES, 2) void paged8_chunk_kernel(AttnArgs a) {
    constexpr int KM = D / 16;           // QK products per 32 keys
    constexpr int DT = D / 32;           // 32-channel tiles of V
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    ChunkLds8<D>& L = *reinterpret_cast<ChunkLds8<D>*>(lds_raw);
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
    const int qe = q_exponent(amax);
    const float qs = pow2(-qe), row_scale = pow2(qe);
    f16x8 qop[KM];
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) qop[m][i] = static_cast<_Float16>(half_at<F16>(qr[m][i >> 1], i & 1) * qs);
    // -128 2^-24 sum(q): what the K codes' offset adds to a score, less it
    float qsum = 0.f;
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) qsum += static_cast<float>(qop[m][i]);
    const auto qh = __builtin_amdgcn_permlane32_swap(__float_as_uint(qsum), __float_as_uint(qsum), false, false);
    const float qbias = -0x1p-17f * (__uint_as_float(qh[0]) + __uint_as_float(qh[1]));
    const int pos = it.len - it.qlen + tok;
    const int lo = first_key(pos, a.window), top = min(pos, it.key1 - 1);
    // every row of this wavefront sees [all_lo, all_hi]
    const int t0 = (it.row0 + min(32 * w, nrows - 1)) / a.G, t1 = (it.row0 + min(32 * w + 31, nrows - 1)) / a.G;
    const int all_hi = min(it.len - it.qlen + t0, it.key1 - 1), all_lo = first_key(it.len - it.qlen + t1, a.window);

    // ---- conversion ----
    // A wavefront has the K and V codes of 8 keys of a block's 64, half a tile: one
    // page id, and descriptors of range 0 (zeros, no access) where the page is not
    // in the pool.
    const int tile = w >> 1;
    const int64_t hk = head * a.ps_head + 8 * (w & 1) * D, hs = head * a.ss_head;
    const int page_mask = (1 << a.page_log2) - 1;
    const int32_t* trow = a.table + it.req * a.bt_stride;
    const int nblk = a.num_pages > 0 ? (max(it.key1 - it.key0, 0) + BLK - 1) / BLK : 0;
    // lane = key * 8 + part: D / 8 codes of K and of V
    constexpr int CODES = D / 32;        // words of them
    const int ckey = lane >> 3, part = lane & 7;
    uint8_t* const kst = L.k[0] + (8 * w + ckey) * KROW<D> + (D / 4) * part;
    uint8_t* const vst = L.v[0] + (8 * w + ckey) * VROW<D> + (D / 4) * part;
    const float *const kscale = static_cast<const float*>(a.ks), *const vscale = static_cast<const float*>(a.vs);
    auto tile_key = [&](int blk) { return it.key0 + BLK * blk + 16 * tile; };
    auto page_id = [&](int blk) -> int { return trow[min(tile_key(blk), it.key1 - 1) >> a.page_log2]; };
    uint32_t kraw[CODES] = {}, vraw[CODES] = {};
    uint32_t ksraw = 0, vsraw = 0;       // scale bits
    bool sok = false;                    // the page is in the pool
    auto fetch = [&](int blk, int id) __attribute__((always_inline)) {
        id = __builtin_amdgcn_readfirstlane(id);
        sok = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_pages);
        const int64_t pg = sok ? id : 0;
        const int o = (min(tile_key(blk), it.key1 - 1) & page_mask) & ~15;
        const int64_t co = pg * a.ps_page + hk + o * D, so = pg * a.ss_page + hs + (o >> 4);
        const Rsrc rk = make_rsrc(a.kp + co, sok ? 8 * D : 0), rv = make_rsrc(a.vp + co, sok ? 8 * D : 0);
        if constexpr (D == 128) {
            const u32x4 k = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, 16 * lane, 0, 0));
            const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, 16 * lane, 0, 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) { kraw[i] = k[i]; vraw[i] = v[i]; }
        } else {
            const u32x2 k = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, 8 * lane, 0, 0));
            const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, 8 * lane, 0, 0));
#pragma unroll
            for (int i = 0; i < 2; ++i) { kraw[i] = k[i]; vraw[i] = v[i]; }
        }
        ksraw = __builtin_amdgcn_raw_buffer_load_b32(make_rsrc(kscale + so, sok ? 4 : 0), 0, 0, 0);
        vsraw = __builtin_amdgcn_raw_buffer_load_b32(make_rsrc(vscale + so, sok ? 4 : 0), 0, 0, 0);
    };
    // the fetched block into buffer b: K as u 2^-24, V as exact codes
    auto store = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < CODES; i += 2) {
            const uint32_t x = kraw[i] ^ FLIP, y = kraw[i + 1] ^ FLIP;
            *reinterpret_cast<u32x4*>(kst + b * static_cast<int>(sizeof(L.k[0])) + 8 * i) = u32x4{bytes2<0>(x), bytes2<2>(x), bytes2<0>(y), bytes2<2>(y)};
        }
#pragma unroll
        for (int i = 0; i < CODES; i += 2) {
            const uint32_t x = vraw[i] ^ FLIP, y = vraw[i + 1] ^ FLIP;
            *reinterpret_cast<u32x4*>(vst + b * static_cast<int>(sizeof(L.v[0])) + 8 * i) = u32x4{codes2<0>(x), codes2<2>(x), codes2<0>(y), codes2<2>(y)};
        }
        if (lane == 0) {                 // (both wavefronts of a tile store the same)
            const float f = checked(__uint_as_float(vsraw));
            L.lv[b][tile] = __builtin_amdgcn_logf(f);
            L.vi[b][tile] = f == f ? __builtin_amdgcn_rcpf(f) : 0.f;
            L.in[b][tile] = sok;
            L.ks[b][tile] = checked(__uint_as_float(ksraw)) * a.scale * 16777216.0f;
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
    // t of half x's keys, and the lane's largest
    auto scores = [&](int b, int x, float m_use) __attribute__((always_inline)) -> float {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float k = L.ks[b][2 * x + i] * row_scale, o = __builtin_fmaf(qbias, k, L.lv[b][2 * x + i] - m_use);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[8 * i + j] = __builtin_fmaf(sc[8 * i + j], k, o);
        }
        float mx = vmax3(t[0], t[1], t[2]);
#pragma unroll
        for (int j = 3; j < 15; j += 2) mx = vmax3(mx, t[j], t[j + 1]);
        return vmax2(mx, t[15]);
    };
    // hides what the rows do not see, and raises their reference where a
    // score passes it
    auto settle = [&](int b, int x, int blk, float mx, float m_use, bool unset) __attribute__((always_inline)) {
        const int j0 = it.key0 + BLK * blk + 32 * x;
        const uint32_t in0 = L.in[b][2 * x], in1 = L.in[b][2 * x + 1];
        if (j0 + 31 > all_hi || j0 < all_lo || !__builtin_amdgcn_readfirstlane(in0 & in1)) {
            mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + 8 * g + 4 * h + i;
                    const bool seen = j <= top && j >= lo && (g < 2 ? in0 : in1);
                    t[4 * g + i] = seen ? t[4 * g + i] : -INFINITY;
                    mx = fmaxf(mx, t[4 * g + i]);
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
    // P' = fp16(2^t) of half x
    auto weights = [&](int b, int x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float ls = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                t[8 * i + j] = fast_exp2(t[8 * i + j]);
                ls += t[8 * i + j];
            }
            l_run = __builtin_fmaf(ls, L.vi[b][2 * x + i], l_run);
#pragma unroll
            for (int j = 0; j < 4; ++j) pw[4 * i + j] = pack_f16x2(t[8 * i + 2 * j], t[8 * i + 2 * j + 1]);
        }
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
        store(0);
        fetch(1, page_id(1));
        store(1);
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
            store(b2);
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
    // registers 4 g .. of a tile are the channels 8 g + 4 h ..
    const int64_t at = (static_cast<int64_t>(it.part) * a.heads + head) * CHUNK + rt;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 o = {acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
            const int ch = 32 * d + 8 * g + 4 * h;
            if (it.part >= 0) *reinterpret_cast<f32x4*>(a.part + at * D + ch) = o;
            else store_row<F16>(a, it.q0, row, head, ch, m_run, l_run, o);
        }
    if (it.part >= 0 && h == 0) { a.ml[at * 2] = m_run; a.ml[at * 2 + 1] = l_run; }
}

template <int D, bool F16>
struct Kernels8 {
    static auto narrow(const AttnArgs& a) { return a.page_log2 > 4 ? paged8_attn_kernel<D, F16, true> : paged8_attn_kernel<D, F16, false>; }
    static constexpr auto chunk = paged8_chunk_kernel<D, F16>;
    static constexpr size_t chunk_lds = sizeof(ChunkLds8<D>);
};

}  // namespace
}  // namespace hyq

using namespace hyq;

extern "C" size_t hyq_paged8_attention_workspace_size(const hyq_paged_params* p) {
    return attention_workspace("hyq_paged8_attention", 4, p);
}

extern "C" int hyq_paged8_attention(const hyq_paged_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    return attention<Kernels8>("hyq_paged8_attention", 4, p, workspace, workspace_bytes, stream);
}
