"""The paged 4-bit KV cache on MI355X: batch layout, append, read-back and
attention over block tables.

The D-stage cache (d_stage_kv_cache.py) holds one batch of equally long
sequences; a program that serves requests of many lengths keeps their K and V
in pages of a common pool instead.  Codes and scales are quantize_per_token's
4-bit rows (hyquant_amd.decode_d_stage):

    k_pages, v_pages  int8 [pages, key heads, page, D / 2]
    k_scale, v_scale  fp16 [pages, key heads, page]

with D 64 or 128 and pages of 16, 32, 64, 128 or 256 tokens.  The pools may be
views into a larger allocation (any page and head strides that keep rows
16-byte aligned; K and V alike).  Token j of request r is row j % page of page
block_table[r, j // page]; its slot is that page's id * page + that row.

A step of a serving program:

    b = paged_batch(context_lens, new_lens, block_table, free_pages, page, num_tokens)
    for each layer:
        paged_append(k, v, b.slots, k_pages, v_pages, k_scale, v_scale)
        out = paged_attention(q, k_pages, v_pages, k_scale, v_scale, block_table, b.seq_lens, b.cu_seqlens)

Nothing is read back to the host, so a captured graph of a step follows the
lengths it is replayed with.  Every call allocates its own outputs and
workspace on the current stream; 256 KiB of arrival counters are kept
per stream of torch's.  Inference only: no gradients.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from . import decode_d_stage as dd
from .decode_d_stage import _HALF, _require_gpu, _stream

PAGE_SIZES = (16, 32, 64, 128, 256)


class PagedBatch(NamedTuple):
    """The layout of one step's batch (paged_batch): parts of one allocation (clone
    one to keep it alone, or to torch.save them together)."""
    cu_seqlens: torch.Tensor      # int32 [R + 1], prefix sums of the new lengths
    seq_lens: torch.Tensor        # int32 [R], context + new
    slots: torch.Tensor           # int64 [num_tokens], -1 past the last new token
    positions: torch.Tensor       # int64 [num_tokens], likewise
    pages_used: torch.Tensor      # int32 [1], pages the step needs


def _fast(t: torch.Tensor):
    """(the C++ form of the calls, t's stream), or (None, 0).  It makes the
    checks below natively and declines whatever fails one (status -1, or the
    library's own status): that call comes back to the Python form, which
    copies what the kernels cannot read, or raises."""
    fx = dd._FX if dd._FX is not None else dd._load_fast_ext()
    if fx and isinstance(t, torch.Tensor) and t.is_cuda:
        return fx, _stream(t.device)
    return None, 0


_counts = {}                               # (device, stream) -> arrival counters of the calls on that stream
_stream_data = getattr(torch._C, "_cuda_getCurrentStream", None)      # (id, device, type)


def _is_torchs(device: torch.device, stream: int) -> bool:
    """Whether the current stream, of handle `stream`, is one of torch's own: one
    that was handed to torch has its handle for an id, torch's have small ones."""
    if _stream_data is not None and device.index is not None:
        return stream == 0 or _stream_data(device.index)[0] != stream
    return stream == 0 or torch.cuda.current_stream(device).stream_id != stream


def _counters(device: torch.device, stream: int) -> int:
    """The address of the arrival counters of eager calls on `stream`, zero
    between calls; 0 while the stream is being captured and has none yet (the
    library uses them in no captured call: a graph may be replayed beside
    eager calls), and for streams that torch does not own: their handles may
    come back for another stream, or name several."""
    c = _counts.get((device.index, stream))
    if c is None:
        if not _is_torchs(device, stream):
            return 0
        with torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                return 0
            c = _counts.setdefault((device.index, stream), torch.zeros(_lib.PAGED_COUNTERS, dtype=torch.int32, device=device))
    return c.data_ptr()


def _ints(t: torch.Tensor, name: str, dtype: torch.dtype, dim: int, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != dim:
        raise ValueError(f"{name} must be a {dim}-d {dtype} tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def _check_page_size(page_size: int) -> None:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page size must be one of {PAGE_SIZES}, got {page_size}")


def _on(device: torch.device):
    """The tensors' device as the current one for the launch."""
    return torch.cuda.device(device)


def paged_batch(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                page_size: int, num_tokens: int) -> PagedBatch:
    """Lay out a step in which request r adds new_lens[r] tokens to its
    context_lens[r] cached ones (int32 [R] each, zeros allowed).

    block_table (int32 [R, max_pages]) is extended in place: the entries of
    the pages that a request newly needs are taken from free_pages (int32),
    in order, request by request; the others are left as they are (its rows
    must not share memory).  num_tokens
    is the length of the token tensors of the step, at least the new tokens'
    sum; the slots and positions behind that sum are -1.  Where free_pages or
    max_pages do not suffice, the missing entries and their tokens' slots are
    -1 (pages_used tells what was needed)."""
    fx, stream = _fast(context_lens)
    if fx:
        try:
            st, *b = fx.paged_batch(context_lens, new_lens, block_table, free_pages, page_size, num_tokens, stream)
            if st == 0:
                return PagedBatch(*b)
        except TypeError:                  # an argument of another type: named below
            pass
    _require_gpu(context_lens, "context_lens")
    dev = context_lens.device
    _ints(context_lens, "context_lens", torch.int32, 1, dev)
    _ints(new_lens, "new_lens", torch.int32, 1, dev)
    _ints(block_table, "block_table", torch.int32, 2, dev)
    _ints(free_pages, "free_pages", torch.int32, 1, dev)
    _check_page_size(page_size)
    R = context_lens.shape[0]
    if new_lens.shape[0] != R or block_table.shape[0] != R:
        raise ValueError(f"context_lens, new_lens and block_table are of {R}, {new_lens.shape[0]} and {block_table.shape[0]} requests")
    if not 0 <= num_tokens < 1 << 31:
        raise ValueError(f"num_tokens must be >= 0 and below 2^31, got {num_tokens}")
    longs = torch.empty(2, num_tokens, dtype=torch.int64, device=dev)
    ints = torch.empty(2 * R + 2, dtype=torch.int32, device=dev)
    cu, lens, used = ints[:R + 1], ints[R + 1:2 * R + 1], ints[2 * R + 1:]
    with _on(dev):
        st = _lib.lib().hyq_paged_batch(
            context_lens.data_ptr(), new_lens.data_ptr(), R, block_table.data_ptr(), block_table.stride(0),
            block_table.shape[1], free_pages.data_ptr(), free_pages.shape[0], page_size, num_tokens, cu.data_ptr(),
            lens.data_ptr(), longs[0].data_ptr(), longs[1].data_ptr(), used.data_ptr(), _stream(dev))
    _lib.check(st, "paged_batch")
    return PagedBatch(cu, lens, longs[0], longs[1], used)


def _check_pool(kp: torch.Tensor, vp: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor, device: torch.device) -> Tuple[int, int, int, int]:
    """(pages, key heads, page size, D) of a pool."""
    for t, name, dtype, dim in ((kp, "k_pages", torch.int8, 4), (vp, "v_pages", torch.int8, 4),
                                (ks, "k_scale", torch.float16, 3), (vs, "v_scale", torch.float16, 3)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != dim:
            raise ValueError(f"{name} must be a {dim}-d {dtype} tensor")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
    N, H, P, DP = kp.shape
    if vp.shape != kp.shape or ks.shape != kp.shape[:3] or vs.shape != kp.shape[:3]:
        raise ValueError(f"k_pages, v_pages, k_scale and v_scale are of shapes {tuple(kp.shape)}, {tuple(vp.shape)}, "
                         f"{tuple(ks.shape)} and {tuple(vs.shape)}")
    _check_page_size(P)
    if DP not in (32, 64):
        raise ValueError(f"head dim must be 64 or 128, got {2 * DP}")
    if N and H:
        if kp.stride() != vp.stride() or ks.stride() != vs.stride():
            raise ValueError("K and V pools must have the same strides")
        if kp.stride(3) != 1 or kp.stride(2) != DP or ks.stride(2) != 1:
            raise ValueError("the rows of a page must be contiguous")
    return N, H, P, 2 * DP


def _pool_args(kp, vp, ks, vs):
    return (kp.data_ptr(), vp.data_ptr(), kp.stride(0), kp.stride(1), ks.data_ptr(), vs.data_ptr(), ks.stride(0),
            ks.stride(1))


def _row_strides(t: torch.Tensor) -> Tuple[int, int]:
    """The strides (token, head) of t [T, H, D]; 0 where there is one alone, whatever t says."""
    return t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous channels and 16-byte aligned rows (a copy if it has others)."""
    if t.numel() and (t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in _row_strides(t))):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _overlaps_itself(t: torch.Tensor) -> bool:
    """Whether rows of t [T, H, D] (contiguous channels) share memory."""
    (n0, n1, D), (s0, s1, _) = t.shape, t.stride()
    if n0 <= 1 or n1 <= 1:
        return (n0 > 1 and s0 < D) or (n1 > 1 and s1 < D)
    return min(s0, s1) < D or (s0 < n1 * s1 and s1 < n0 * s0)


def paged_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Quantise the rows k, v [T, H, D] (bf16 or fp16, any strides) into their
    slots (int64 [T]): bit for bit quantize_per_token's codes and scales.  A
    slot outside the pool writes nothing; the slots of one call have to be
    distinct."""
    fx, stream = _fast(k)
    if fx:
        try:
            if fx.paged_append(k, v, slots, k_pages, v_pages, k_scale, v_scale, stream) == 0:
                return
        except TypeError:
            pass
    _require_gpu(k, "k")
    N, H, P, D = _check_pool(k_pages, v_pages, k_scale, v_scale, k.device)
    if k.dtype not in _HALF or v.dtype != k.dtype:
        raise ValueError(f"paged_append expects bf16 or fp16 rows of one dtype, got {k.dtype} and {v.dtype}")
    if k.dim() != 3 or k.shape != v.shape or tuple(k.shape[1:]) != (H, D):
        raise ValueError(f"k and v must be [T, {H}, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if v.device != k.device:
        raise ValueError(f"v is on {v.device}, not on {k.device}")
    _ints(slots, "slots", torch.int64, 1, k.device)
    if slots.shape[0] != k.shape[0]:
        raise ValueError(f"{slots.shape[0]} slots for {k.shape[0]} rows")
    k, v = _aligned_rows(k), _aligned_rows(v)
    with _on(k.device):
        st = _lib.lib().hyq_paged_append(
            k.data_ptr(), *_row_strides(k), v.data_ptr(), *_row_strides(v), int(k.dtype == torch.float16),
            slots.data_ptr(), k.shape[0], H, D, *_pool_args(k_pages, v_pages, k_scale, v_scale), N, P, _stream(k.device))
    _lib.check(st, "paged_append")


def paged_gather(slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows [T, H, D] of slots (int64 [T]) as bf16 or fp16: code *
    scale rounded once; zeros for slots outside the pool."""
    fx, stream = _fast(slots)
    if fx and dtype in _HALF:
        try:
            st, k, v = fx.paged_gather(slots, k_pages, v_pages, k_scale, v_scale, dtype == torch.float16, stream)
            if st == 0:
                return k, v
        except TypeError:
            pass
    _require_gpu(slots, "slots")
    _ints(slots, "slots", torch.int64, 1, slots.device)
    N, H, P, D = _check_pool(k_pages, v_pages, k_scale, v_scale, slots.device)
    if dtype not in _HALF:
        raise ValueError(f"paged_gather gives bf16 or fp16 rows, not {dtype}")
    T = slots.shape[0]
    k, v = (torch.empty(T, H, D, dtype=dtype, device=slots.device) for _ in range(2))
    with _on(slots.device):
        st = _lib.lib().hyq_paged_gather(slots.data_ptr(), T, H, D, *_pool_args(k_pages, v_pages, k_scale, v_scale), N, P,
                                         int(dtype == torch.float16), k.data_ptr(), v.data_ptr(), _stream(slots.device))
    _lib.check(st, "paged_gather")
    return k, v


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    cu_seqlens: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None, window: int = 0,
                    return_lse: bool = False,
                    out: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of the new tokens of R requests over their cached
    tokens (their own among them: append first).

    q [T, H_Q, D] bf16 or fp16, H_Q a multiple of the pool's key heads.
    Request r has the tokens [cu_seqlens[r], cu_seqlens[r + 1]) (int32 [R + 1]
    from 0); without cu_seqlens, a decode step, token r alone (T = R).  They
    are the last of its seq_lens[r] (int32 [R]) tokens: a token at position p
    sees the keys j <= p, with window > 0 only the last `window` of those.

    Returns out [T, H_Q, D] of q's dtype, with return_lse also the natural
    log-sum-exp of the scaled scores, fp32 [T, H_Q].  A row that sees no key is
    zero (lse -inf), as are the rows behind the last request of a padded batch
    (those of an `out` that is handed in are left as they are; it shares no
    memory with the inputs)."""
    fx, stream = _fast(q)
    if fx and out is None:
        try:
            st, o, lse = fx.paged_attention(q, k_pages, v_pages, k_scale, v_scale, block_table, seq_lens, cu_seqlens,
                                            sm_scale, window, return_lse, stream, 0 if cu_seqlens is not None else _counters(q.device, stream))
            if st == 0:
                return (o, lse) if return_lse else o
        except TypeError:
            pass
    _require_gpu(q, "q")
    dev = q.device
    N, H, P, D = _check_pool(k_pages, v_pages, k_scale, v_scale, dev)
    if q.dtype not in _HALF:
        raise ValueError(f"paged_attention expects bf16 or fp16 queries, got {q.dtype}")
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q must be [T, H_Q, {D}], got {tuple(q.shape)}")
    T, HQ, _ = q.shape
    if H == 0 or HQ == 0 or HQ % H:
        raise ValueError(f"{HQ} query heads are no multiple of {H} key heads")
    _ints(block_table, "block_table", torch.int32, 2, dev)
    _ints(seq_lens, "seq_lens", torch.int32, 1, dev)
    R = seq_lens.shape[0]
    if block_table.shape[0] != R:
        raise ValueError(f"block_table and seq_lens are of {block_table.shape[0]} and {R} requests")
    if cu_seqlens is None:
        if T != R:
            raise ValueError(f"{T} tokens of {R} requests need cu_seqlens")
    else:
        _ints(cu_seqlens, "cu_seqlens", torch.int32, 1, dev)
        if cu_seqlens.shape[0] != R + 1:
            raise ValueError(f"cu_seqlens must be of {R + 1} entries, got {cu_seqlens.shape[0]}")
    if window < 0:
        raise ValueError(f"window must be >= 0, got {window}")
    window = window if window < 1 << 30 else 0       # (no table row names as many tokens)
    zero_tail = out is None
    if out is None:
        out = torch.empty(T, HQ, D, dtype=q.dtype, device=dev)
    elif out.dtype != q.dtype or out.shape != q.shape or out.device != dev or out.stride(2) != 1:
        raise ValueError("out must be of q's shape, dtype and device, with contiguous channels")
    elif _overlaps_itself(out) or (T and out.data_ptr() == q.data_ptr()):
        raise ValueError("out must not share memory between its rows, or with q")
    lse = torch.empty(T, HQ, dtype=torch.float32, device=dev) if return_lse else None
    if T and R:
        q = _aligned_rows(q)
        p = _lib.PagedParams()
        p.q, (p.q_stride_t, p.q_stride_h) = q.data_ptr(), _row_strides(q)
        p.out, (p.o_stride_t, p.o_stride_h) = out.data_ptr(), _row_strides(out)
        p.lse = lse.data_ptr() if return_lse else None
        (p.k_pages, p.v_pages, p.p_stride_page, p.p_stride_head, p.k_scale, p.v_scale, p.s_stride_page,
         p.s_stride_head) = _pool_args(k_pages, v_pages, k_scale, v_scale)
        p.block_table, p.bt_stride = block_table.data_ptr(), block_table.stride(0)
        p.seq_lens, p.cu_seqlens = seq_lens.data_ptr(), None if cu_seqlens is None else cu_seqlens.data_ptr()
        p.num_pages, p.page_size, p.max_pages, p.num_requests, p.num_tokens = N, P, block_table.shape[1], R, T
        p.kv_heads, p.kv_repeat, p.head_dim, p.window = H, HQ // H, D, window
        p.sm_scale = D ** -0.5 if sm_scale is None else sm_scale
        p.dtype_fp16, p.zero_tail = int(q.dtype == torch.float16), 3 if zero_tail else 2
        if cu_seqlens is None:
            p.counters = _counters(dev, _stream(dev)) or None
        L = _lib.lib()
        ref = ctypes.byref(p)
        need = L.hyq_paged_attention_workspace_size(ref)
        # a workspace of its own for every call: two streams or captured graphs never share one
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        with _on(dev):
            st = L.hyq_paged_attention(ref, ws.data_ptr(), need, _stream(dev))
        _lib.check(st, "paged_attention")
    elif T:                                # no request: every row is behind the last
        if zero_tail:
            out.zero_()
        if return_lse:
            lse.fill_(float("-inf"))
    return (out, lse) if return_lse else out
