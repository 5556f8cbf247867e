// Eager fast paths of a decode step: fused_d_stage_decode
// (src/ops/decode_d_stage.py:470-1005 is the reference's call), the same over
// a layer cache's own buffers, and its staging append
// (src/ops/d_stage_kv_cache.py:195-207).  A Python extension that reads the
// tensors' metadata natively, fills one hyq_decode_params, allocates the
// output and calls hyq_decode_hybrid through the pointer the Python side
// hands over at set-up (the library ctypes loaded, whichever file that is).
//
// The paged cache's calls (hyquant_amd/paged.py) take the same way: each makes
// the checks of its Python form and declines (status -1) whatever fails one,
// so that the Python form copies, or raises.
//
// decode takes exactly the calls the Python fast path takes (bf16 / fp16 q
// with unit channel stride, kv_repeat dividing the query heads, CUDA tensors,
// the three bf16 segments with unit channel strides, equal K / V lengths and
// one dtype, the quantised prefix with unit innermost strides); decode_cache
// the same over a cache's buffers, with q's heads one stride apart; append
// plain CUDA rows of the buffers' type and device that autograd does not
// record.  Anything else returns status -1 and the caller takes its other
// paths (the checked call, two tensor copies).  The library
// validates every field (alignment, 32-bit strides, sizes) before it
// launches, as for every other caller.  Host code only: no kernel here.

#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <optional>

#include "../../include/hyq.h"

namespace {

using HybridFn = int (*)(const hyq_decode_params*, void*, size_t, void*);
HybridFn g_hybrid = nullptr;
using AppendFn = decltype(&hyq_append_rows);
AppendFn g_append = nullptr;

// The first n rows (all of them: n < 0) of one bf16 / fp16 segment: 0 empty,
// 1 bf16, 2 fp16, -1 not taken
int segment(const at::Tensor& k, const at::Tensor& v, hyq_decode_params& p, int s, int64_t n = -1) {
    if (k.dim() != 3 || v.dim() != 3) return -1;
    if (v.size(1) != k.size(1) || n > k.size(1)) return k.size(1) == 0 && n <= 0 ? 0 : -1;
    if (n < 0) n = k.size(1);
    if (n == 0) return 0;
    const auto dt = k.scalar_type();
    if (k.stride(2) != 1 || v.stride(2) != 1 || v.scalar_type() != dt) return -1;
    if (dt != at::kBFloat16 && dt != at::kHalf) return -1;
    p.seg_k[s] = static_cast<const uint16_t*>(k.data_ptr());
    p.seg_k_stride_bh[s] = k.stride(0);
    p.seg_k_stride_n[s] = k.stride(1);
    p.seg_v[s] = static_cast<const uint16_t*>(v.data_ptr());
    p.seg_v_stride_bh[s] = v.stride(0);
    p.seg_v_stride_n[s] = v.stride(1);
    p.seg_n[s] = n;
    return dt == at::kBFloat16 ? 1 : 2;
}

using Result = std::tuple<int64_t, at::Tensor>;

// q: query rows of d channels, q_stride apart; nq and ns: the tokens of the
// prefix and of the staging segment (-1: the tensors' own); out_shape: the
// shape of the returned tensor (contiguous, bh_q * d values)
Result run(const at::Tensor& q, int64_t bh_q, int64_t d, int64_t q_stride, at::IntArrayRef out_shape,
           const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks, const at::Tensor& vs, int64_t nq,
           const at::Tensor& kt, const at::Tensor& vt, const at::Tensor& kst, const at::Tensor& vst, int64_t ns,
           const at::Tensor& kw, const at::Tensor& vw, int64_t k_bits, int64_t v_bits, int64_t kv_repeat,
           double sm_scale, int64_t split_tokens, int64_t stream, int64_t ws, int64_t ws_bytes) {
    const Result skip{-1, at::Tensor()};
    hyq_decode_params p{};
    const auto qdt = q.scalar_type();
    if (qdt == at::kBFloat16) p.dtype_flags = 0;
    else if (qdt == at::kHalf) p.dtype_flags = HYQ_DT_Q_FP16 | HYQ_DT_OUT_FP16;
    else return skip;
    if (kv_repeat < 1 || bh_q % kv_repeat) return skip;
    int dts = 0;
    const at::Tensor* segs[3][2] = {{&kt, &vt}, {&kst, &vst}, {&kw, &vw}};
    for (int s = 0; s < 3; ++s) {
        const int dt = segment(*segs[s][0], *segs[s][1], p, s, s == 1 ? ns : -1);
        if (dt < 0) return skip;
        if (dt > 0) {
            if (dts && dts != dt) return skip;
            dts = dt;
        }
    }
    if (dts == 2) p.dtype_flags |= HYQ_DT_SEG_FP16;
    if (kp.dim() != 3 || vp.dim() != 3 || ks.dim() != 2 || vs.dim() != 2) return skip;
    if (nq < 0) nq = kp.size(1);
    if (nq > kp.size(1)) return skip;
    if (nq > 0) {
        if (kp.stride(2) != 1 || vp.stride(2) != 1 || ks.stride(1) != 1 || vs.stride(1) != 1) return skip;
        p.k_packed = static_cast<const int8_t*>(kp.data_ptr());
        p.kp_stride_bh = kp.stride(0);
        p.kp_stride_n = kp.stride(1);
        p.v_packed = static_cast<const int8_t*>(vp.data_ptr());
        p.vp_stride_bh = vp.stride(0);
        p.vp_stride_n = vp.stride(1);
        p.k_scale = static_cast<const uint16_t*>(ks.data_ptr());
        p.ks_stride_bh = ks.stride(0);
        p.v_scale = static_cast<const uint16_t*>(vs.data_ptr());
        p.vs_stride_bh = vs.stride(0);
    }
    p.n_quant = nq;
    at::Tensor out = at::empty(out_shape, q.options());
    p.q = static_cast<const uint16_t*>(q.data_ptr());
    p.q_stride = q_stride;
    p.out = static_cast<uint16_t*>(out.data_ptr());
    p.out_stride = d;
    p.bh_kv = static_cast<int32_t>(bh_q / kv_repeat);
    p.kv_repeat = static_cast<int32_t>(kv_repeat);
    p.head_dim = static_cast<int32_t>(d);
    p.k_bits = static_cast<int32_t>(k_bits);
    p.v_bits = static_cast<int32_t>(v_bits);
    // (head_dim ** -0.5 as Python computes it, then rounded to float)
    p.sm_scale = std::isnan(sm_scale) ? static_cast<float>(std::pow(static_cast<double>(d), -0.5))
                                      : static_cast<float>(sm_scale);
    p.split_tokens = static_cast<int32_t>(split_tokens);
    const int st = g_hybrid(&p, reinterpret_cast<void*>(ws), static_cast<size_t>(ws_bytes),
                            reinterpret_cast<void*>(stream));
    return {st, out};
}

// ---- the paged cache ---------------------------------------------------------

using BatchFn = decltype(&hyq_paged_batch);
using PagedAppendFn = decltype(&hyq_paged_append);
using GatherFn = decltype(&hyq_paged_gather);
using AttentionFn = decltype(&hyq_paged_attention);
using AttentionSizeFn = decltype(&hyq_paged_attention_workspace_size);
struct {
    BatchFn batch = nullptr;
    PagedAppendFn append = nullptr;
    GatherFn gather = nullptr;
    AttentionSizeFn size = nullptr;
    AttentionFn attention = nullptr;
} g_paged;

bool plain(const at::Tensor& t, at::ScalarType type, int64_t dim, const at::Device& device) {
    return t.scalar_type() == type && t.dim() == dim && t.device() == device && !at::isTensorSubclassLike(t);
}
// an integer tensor whose last dimension is contiguous
bool ints(const at::Tensor& t, at::ScalarType type, int64_t dim, const at::Device& device) {
    return plain(t, type, dim, device) && (t.stride(dim - 1) == 1 || t.numel() <= 1);
}
bool half(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
// rows of channels at 16-byte addresses
bool rows16(const at::Tensor& t) {
    return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
           reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
// a pool as _check_pool wants it (sizes and alignment are the library's to check)
bool pool(const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks, const at::Tensor& vs, const at::Device& device) {
    if (!plain(kp, at::kChar, 4, device) || !plain(vp, at::kChar, 4, device) || !plain(ks, at::kHalf, 3, device) ||
        !plain(vs, at::kHalf, 3, device))
        return false;
    if (kp.sizes() != vp.sizes() || kp.strides() != vp.strides() || ks.sizes() != vs.sizes() || ks.strides() != vs.strides())
        return false;
    if (ks.size(0) != kp.size(0) || ks.size(1) != kp.size(1) || ks.size(2) != kp.size(2)) return false;
    return kp.numel() > 0 && kp.stride(3) == 1 && kp.stride(2) == kp.size(3) && ks.stride(2) == 1;
}
template <typename T>
T* ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

// A contiguous tensor of `type` at element `offset` of base's memory.  A call's
// outputs are parts of one allocation this way: an allocation costs about 0.6 us
// of host time, a part about 0.1.
at::Tensor part(const at::Tensor& base, at::ScalarType type, int64_t offset, at::IntArrayRef sizes) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
}

}  // namespace

void set_paged(int64_t batch, int64_t append, int64_t gather, int64_t size, int64_t attention) {
    g_paged.batch = reinterpret_cast<BatchFn>(batch);
    g_paged.append = reinterpret_cast<PagedAppendFn>(append);
    g_paged.gather = reinterpret_cast<GatherFn>(gather);
    g_paged.size = reinterpret_cast<AttentionSizeFn>(size);
    g_paged.attention = reinterpret_cast<AttentionFn>(attention);
}

// (status, cu_seqlens, seq_lens, slots, positions, pages_used)
std::tuple<int64_t, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> paged_batch(
    const at::Tensor& ctx, const at::Tensor& fresh, const at::Tensor& table, const at::Tensor& free_pages, int64_t page,
    int64_t tokens, int64_t stream) {
    const auto dev = ctx.device();
    const int64_t R = ctx.dim() == 1 ? ctx.size(0) : 0;
    if (!g_paged.batch || !dev.is_cuda() || R < 1 || tokens < 0 || tokens > INT32_MAX || page < 0 || page > INT32_MAX ||
        !ints(ctx, at::kInt, 1, dev) || !ints(fresh, at::kInt, 1, dev) || !ints(table, at::kInt, 2, dev) ||
        !ints(free_pages, at::kInt, 1, dev) || fresh.size(0) != R || table.size(0) != R || free_pages.size(0) > INT32_MAX)
        return {-1, {}, {}, {}, {}, {}};
    const c10::DeviceGuard guard(dev);
    // slots, positions, then (in halves of a word) offsets, lengths and the count
    const at::Tensor all = at::empty({2 * tokens + R + 1}, ctx.options().dtype(at::kLong));
    const int64_t ints_at = 4 * tokens;
    const at::Tensor slots = part(all, at::kLong, 0, {tokens}), positions = part(all, at::kLong, tokens, {tokens});
    const at::Tensor cu = part(all, at::kInt, ints_at, {R + 1}), lens = part(all, at::kInt, ints_at + R + 1, {R}), used = part(all, at::kInt, ints_at + 2 * R + 1, {1});
    const int st = g_paged.batch(ptr<int32_t>(ctx), ptr<int32_t>(fresh), static_cast<int32_t>(R), ptr<int32_t>(table), table.stride(0),
                                 static_cast<int32_t>(table.size(1)), ptr<int32_t>(free_pages),
                                 static_cast<int32_t>(free_pages.size(0)), static_cast<int32_t>(page), static_cast<int32_t>(tokens),
                                 ptr<int32_t>(cu), ptr<int32_t>(lens), ptr<int64_t>(slots), ptr<int64_t>(positions),
                                 ptr<int32_t>(used), reinterpret_cast<void*>(stream));
    return {st, cu, lens, slots, positions, used};
}

int64_t paged_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots, const at::Tensor& kp, const at::Tensor& vp,
                     const at::Tensor& ks, const at::Tensor& vs, int64_t stream) {
    const auto dev = k.device();
    if (!g_paged.append || !dev.is_cuda() || !half(k) || !plain(k, k.scalar_type(), 3, dev) || !plain(v, k.scalar_type(), 3, dev) ||
        k.sizes() != v.sizes() || !pool(kp, vp, ks, vs, dev) || k.size(1) != kp.size(1) || k.size(2) != 2 * kp.size(3) ||
        !ints(slots, at::kLong, 1, dev) || slots.size(0) != k.size(0) || k.size(0) == 0 || !rows16(k) || !rows16(v))
        return -1;
    const c10::DeviceGuard guard(dev);
    return g_paged.append(ptr<uint16_t>(k), k.stride(0), k.stride(1), ptr<uint16_t>(v), v.stride(0), v.stride(1),
                          k.scalar_type() == at::kHalf, ptr<int64_t>(slots), k.size(0), static_cast<int32_t>(kp.size(1)),
                          static_cast<int32_t>(k.size(2)), ptr<int8_t>(kp), ptr<int8_t>(vp), kp.stride(0), kp.stride(1),
                          ptr<uint16_t>(ks), ptr<uint16_t>(vs), ks.stride(0), ks.stride(1), kp.size(0),
                          static_cast<int32_t>(kp.size(2)), reinterpret_cast<void*>(stream));
}

// (status, k, v)
std::tuple<int64_t, at::Tensor, at::Tensor> paged_gather(const at::Tensor& slots, const at::Tensor& kp, const at::Tensor& vp,
                                                         const at::Tensor& ks, const at::Tensor& vs, bool fp16, int64_t stream) {
    const auto dev = slots.device();
    if (!g_paged.gather || !dev.is_cuda() || !ints(slots, at::kLong, 1, dev) || slots.size(0) == 0 || !pool(kp, vp, ks, vs, dev))
        return {-1, {}, {}};
    const c10::DeviceGuard guard(dev);
    const auto opt = slots.options().dtype(fp16 ? at::kHalf : at::kBFloat16);
    const at::Tensor kv = at::empty({2, slots.size(0), kp.size(1), 2 * kp.size(3)}, opt);
    const at::Tensor k = part(kv, kv.scalar_type(), 0, kv.sizes().slice(1));
    const at::Tensor v = part(kv, kv.scalar_type(), k.numel(), kv.sizes().slice(1));
    const int st = g_paged.gather(ptr<int64_t>(slots), slots.size(0), static_cast<int32_t>(kp.size(1)),
                                  static_cast<int32_t>(2 * kp.size(3)), ptr<int8_t>(kp), ptr<int8_t>(vp), kp.stride(0), kp.stride(1),
                                  ptr<uint16_t>(ks), ptr<uint16_t>(vs), ks.stride(0), ks.stride(1), kp.size(0),
                                  static_cast<int32_t>(kp.size(2)), fp16, ptr<uint16_t>(k), ptr<uint16_t>(v),
                                  reinterpret_cast<void*>(stream));
    return {st, k, v};
}

// (status, out, lse)
std::tuple<int64_t, at::Tensor, at::Tensor> paged_attention(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp,
                                                            const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                                                            const at::Tensor& lens, const std::optional<at::Tensor>& cu,
                                                            const std::optional<double>& sm_scale, int64_t window,
                                                            bool want_lse, int64_t stream, int64_t counters) {
    const std::tuple<int64_t, at::Tensor, at::Tensor> skip{-1, {}, {}};
    const auto dev = q.device();
    if (!g_paged.attention || !dev.is_cuda() || !half(q) || !plain(q, q.scalar_type(), 3, dev) || !pool(kp, vp, ks, vs, dev) ||
        !ints(table, at::kInt, 2, dev) || !ints(lens, at::kInt, 1, dev))
        return skip;
    const int64_t T = q.size(0), HQ = q.size(1), D = q.size(2), R = lens.size(0), H = kp.size(1);
    if (T == 0 || R == 0 || T > INT32_MAX || HQ == 0 || HQ % H || D != 2 * kp.size(3) || table.size(0) != R || !rows16(q) || window < 0 ||
        window > INT32_MAX)
        return skip;
    if (cu ? !ints(*cu, at::kInt, 1, dev) || cu->size(0) != R + 1 : T != R) return skip;
    const c10::DeviceGuard guard(dev);
    const at::Tensor out = at::empty({T, HQ, D}, q.options());
    at::Tensor lse;
    hyq_paged_params p{};
    if (want_lse) {
        lse = at::empty({T, HQ}, q.options().dtype(at::kFloat));
        p.lse = ptr<float>(lse);
    }
    p.q = q.data_ptr();
    p.q_stride_t = q.stride(0);
    p.q_stride_h = q.stride(1);
    p.out = out.data_ptr();
    p.o_stride_t = HQ * D;
    p.o_stride_h = D;
    p.k_pages = ptr<int8_t>(kp);
    p.v_pages = ptr<int8_t>(vp);
    p.p_stride_page = kp.stride(0);
    p.p_stride_head = kp.stride(1);
    p.k_scale = ptr<uint16_t>(ks);
    p.v_scale = ptr<uint16_t>(vs);
    p.s_stride_page = ks.stride(0);
    p.s_stride_head = ks.stride(1);
    p.block_table = ptr<int32_t>(table);
    p.bt_stride = table.stride(0);
    p.seq_lens = ptr<int32_t>(lens);
    p.cu_seqlens = cu ? ptr<int32_t>(*cu) : nullptr;
    p.num_pages = kp.size(0);
    p.page_size = static_cast<int32_t>(kp.size(2));
    p.max_pages = static_cast<int32_t>(table.size(1));
    p.num_requests = static_cast<int32_t>(R);
    p.num_tokens = static_cast<int32_t>(T);
    p.kv_heads = static_cast<int32_t>(H);
    p.kv_repeat = static_cast<int32_t>(HQ / H);
    p.head_dim = static_cast<int32_t>(D);
    p.window = static_cast<int32_t>(window);
    p.sm_scale = static_cast<float>(sm_scale ? *sm_scale : std::pow(static_cast<double>(D), -0.5));
    p.dtype_fp16 = q.scalar_type() == at::kHalf;
    p.zero_tail = 3;
    p.counters = reinterpret_cast<uint32_t*>(counters);
    const size_t need = g_paged.size(&p);
    if (need == 0) return skip;
    const at::Tensor ws = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
    const int st = g_paged.attention(&p, ws.data_ptr(), need, reinterpret_cast<void*>(stream));
    return {st, out, lse};
}

// the paged parameter block's size and the offsets of two of its fields
std::tuple<int64_t, int64_t, int64_t> paged_layout() {
    return {static_cast<int64_t>(sizeof(hyq_paged_params)), static_cast<int64_t>(offsetof(hyq_paged_params, num_pages)),
            static_cast<int64_t>(offsetof(hyq_paged_params, counters))};
}

// the library entry points (addresses from ctypes)
void set_entry(int64_t hybrid, int64_t append) {
    g_hybrid = reinterpret_cast<HybridFn>(hybrid);
    g_append = reinterpret_cast<AppendFn>(append);
}

// (status, out): status 0 launched; -1 not taken (nothing launched); any
// other value is the library's status for this call (nothing launched)
Result decode(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks,
              const at::Tensor& vs, const at::Tensor& kt, const at::Tensor& vt, const at::Tensor& kst,
              const at::Tensor& vst, const at::Tensor& kw, const at::Tensor& vw, int64_t k_bits, int64_t v_bits,
              int64_t kv_repeat, double sm_scale, int64_t split_tokens, int64_t stream, int64_t ws, int64_t ws_bytes) {
    if (!g_hybrid || q.dim() != 2 || !q.is_cuda() || q.stride(1) != 1) return {-1, at::Tensor()};
    return run(q, q.size(0), q.size(1), q.stride(0), {q.size(0), q.size(1)}, kp, vp, ks, vs, -1, kt, vt, kst, vst, -1,
               kw, vw, k_bits, v_bits, kv_repeat, sm_scale, split_tokens, stream, ws, ws_bytes);
}

// One layer's decode step over its cache's own buffers: q [b, hq, 1, d] of the
// cache's batch, the first nq tokens of the prefix store, the first ns rows of
// the staging buffers.  Returns [b, hq, 1, d].
Result decode_cache(const at::Tensor& q, int64_t batch, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks,
                    const at::Tensor& vs, int64_t nq, const at::Tensor& kt, const at::Tensor& vt, const at::Tensor& kst,
                    const at::Tensor& vst, int64_t ns, const at::Tensor& kw, const at::Tensor& vw, int64_t k_bits,
                    int64_t v_bits, int64_t kv_repeat, int64_t stream, int64_t ws, int64_t ws_bytes) {
    const Result skip{-1, at::Tensor()};
    if (!g_hybrid || q.dim() != 4 || !q.is_cuda() || nq < 0 || ns < 0) return skip;
    const int64_t b = q.size(0), h = q.size(1), d = q.size(3);
    // the rows of all heads have to be one stride apart
    if (q.size(2) != 1 || q.stride(3) != 1 || b * h * d == 0 || (h > 1 && b > 1 && q.stride(0) != h * q.stride(1)))
        return skip;
    if (b != batch || kt.size(0) * kv_repeat != b * h) return skip;
    const int64_t row = h > 1 ? q.stride(1) : b > 1 ? q.stride(0) : d;
    return run(q, b * h, d, row, {b, h, 1, d}, kp, vp, ks, vs, nq, kt, vt, kst, vst, ns, kw, vw, k_bits, v_bits,
               kv_repeat, std::nan(""), 0, stream, ws, ws_bytes);
}

// Rows of k and v [b, h, n, d] into staging buffers [b * h, cap, d] at `row`.
// Status 0 launched, -1 not taken (nothing written), else the library's.
int64_t append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& dk, const at::Tensor& dv, int64_t row,
               int64_t stream) {
    if (!g_append || k.dim() != 4 || dk.dim() != 3 || !k.is_cuda() || !v.is_cuda()) return -1;
    if (k.sizes() != v.sizes() || dk.sizes() != dv.sizes() || dk.strides() != dv.strides()) return -1;
    if (k.scalar_type() != dk.scalar_type() || v.scalar_type() != dk.scalar_type() || dv.scalar_type() != dk.scalar_type())
        return -1;
    if (k.device() != dk.device() || v.device() != dk.device() || dk.element_size() != 2) return -1;
    // a copy that autograd records, or a tensor that is not plain memory, goes to copy_
    if (at::GradMode::is_enabled() && (k.requires_grad() || v.requires_grad())) return -1;
    if (k.is_conj() || v.is_conj() || k.is_neg() || v.is_neg()) return -1;
    if (at::isTensorSubclassLike(k) || at::isTensorSubclassLike(v)) return -1;
    const int64_t n = k.size(2), d = k.size(3);
    if (k.size(0) * k.size(1) != dk.size(0) || d != dk.size(2) || row < 0 || row + n > dk.size(1)) return -1;
    if (k.stride(3) != 1 || v.stride(3) != 1 || dk.stride(2) != 1 || dk.stride(1) != d) return -1;
    const c10::DeviceGuard guard(k.device());             // as copy_ does
    return g_append(static_cast<const uint16_t*>(k.data_ptr()), k.stride(0), k.stride(1), k.stride(2),
                    static_cast<const uint16_t*>(v.data_ptr()), v.stride(0), v.stride(1), v.stride(2),
                    static_cast<int32_t>(k.size(0)), static_cast<int32_t>(k.size(1)), n, static_cast<int32_t>(d),
                    static_cast<uint16_t*>(dk.data_ptr()), static_cast<uint16_t*>(dv.data_ptr()), dk.stride(0), row,
                    reinterpret_cast<void*>(stream));
}

// the parameter block's size and the offsets of its first and last fields,
// which the caller compares with its own view of include/hyq.h before it
// uses this module
std::tuple<int64_t, int64_t, int64_t> layout() {
    return {static_cast<int64_t>(sizeof(hyq_decode_params)),
            static_cast<int64_t>(offsetof(hyq_decode_params, seg_n)),
            static_cast<int64_t>(offsetof(hyq_decode_params, dtype_flags))};
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("signatures", [] { return 4; }, "counts up when a function of this module takes other arguments");
    m.def("layout", &layout, "sizeof(hyq_decode_params), offsetof(seg_n), offsetof(dtype_flags)");
    m.def("set_entry", &set_entry, "the addresses of hyq_decode_hybrid and hyq_append_rows");
    m.def("decode", &decode, "fused_d_stage_decode eager fast path");
    m.def("decode_cache", &decode_cache, "a layer cache's decode step");
    m.def("append", &append, "a layer cache's staging append");
    m.def("paged_layout", &paged_layout, "sizeof(hyq_paged_params), offsetof(num_pages), offsetof(counters)");
    m.def("set_paged", &set_paged, "the addresses of the five hyq_paged entry points");
    m.def("paged_batch", &paged_batch, "a step's batch layout");
    m.def("paged_append", &paged_append, "new rows into the pages");
    m.def("paged_gather", &paged_gather, "rows of the pages");
    m.def("paged_attention", &paged_attention, "attention over the pages");
}
