"""The paged 8-bit KV cache on MI355X: append, read-back and attention over block
tables.

The sibling of the 4-bit cache of hyquant_amd.paged for programs that want its
pages with less loss: int8 codes and one scale, a power of two, for each block of
16 tokens and key head,

    k_pages, v_pages  int8 [pages, key heads, page, D]
    k_scale, v_scale  fp32 [pages, key heads, page / 16]      value = code * scale

with D 64 or 128 and pages of 16, 32, 64, 128 or 256 tokens; strides, block
tables and slots as there, and paged_batch lays out its steps too.

A block's scale is the smallest 2^e with max(|x|, 1e-5) <= 127 * 2^e.  Tokens
that join a block may raise it: the codes of the tokens that are there are then
rounded again, code * old / new, so that a value is off by at most one step of
the block's last scale.  Inference only: no gradients.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .decode_d_stage import _HALF, _require_gpu, _stream
from .paged import _aligned_rows, _attend, _check_page_size, _fast, _ints, _on, _row_strides

SCALE_BLOCK = 16                           # tokens of a scale


def _check_pool8(kp: torch.Tensor, vp: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor, device: torch.device) -> Tuple[int, int, int, int]:
    """(pages, key heads, page size, D) of an 8-bit pool."""
    for t, name, dtype, dim in ((kp, "k_pages", torch.int8, 4), (vp, "v_pages", torch.int8, 4),
                                (ks, "k_scale", torch.float32, 3), (vs, "v_scale", torch.float32, 3)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != dim:
            raise ValueError(f"{name} must be a {dim}-d {dtype} tensor")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
    N, H, P, D = kp.shape
    _check_page_size(P)
    if vp.shape != kp.shape or tuple(ks.shape) != (N, H, P // SCALE_BLOCK) or ks.shape != vs.shape:
        raise ValueError(f"k_pages, v_pages, k_scale and v_scale are of shapes {tuple(kp.shape)}, {tuple(vp.shape)}, "
                         f"{tuple(ks.shape)} and {tuple(vs.shape)}")
    if D not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, got {D}")
    if N and H:
        if kp.stride() != vp.stride() or ks.stride() != vs.stride():
            raise ValueError("K and V pools must have the same strides")
        if kp.stride(3) != 1 or kp.stride(2) != D or (P > SCALE_BLOCK and ks.stride(2) != 1):
            raise ValueError("the rows of a page must be contiguous")
    return N, H, P, D


def _pool_struct(kp, vp, ks, vs, bits: int) -> "_lib.PagedPool":
    return _lib.PagedPool(kp.data_ptr(), vp.data_ptr(), kp.stride(0), kp.stride(1), ks.data_ptr(), vs.data_ptr(), ks.stride(0),
                          ks.stride(1), kp.shape[0], kp.shape[2], bits)


def paged8_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                  k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Put the rows k, v [T, H, D] (bf16 or fp16, any strides) into their slots
    (int64 [T]).  A slot outside the pool writes nothing, wherever it stands.  The
    slots of one call are distinct, those of one block of 16 are neighbours (but for
    slots outside the pool) and ascend, as paged_batch gives them, and the rows of a
    block before its first new one were appended by earlier calls; rows behind its
    last new one hold anything after the call.  A block with a value that is not
    finite, or past 127 * 2^40, has the scale NaN for as long as earlier rows of it
    stay; their codes are untouched.

    A scale does not fall by itself.  Tokens that are taken back (a rejected draft)
    have coarsened the block that they share with accepted ones, or made its scale
    NaN: put its codes and scales back as they were before, or append its tokens
    again from its first slot on."""
    fx, stream = _fast(k)
    if fx:
        try:
            if fx.paged8_append(k, v, slots, k_pages, v_pages, k_scale, v_scale, stream) == 0:
                return
        except TypeError:
            pass
    _require_gpu(k, "k")
    N, H, P, D = _check_pool8(k_pages, v_pages, k_scale, v_scale, k.device)
    if k.dtype not in _HALF or v.dtype != k.dtype:
        raise ValueError(f"paged8_append expects bf16 or fp16 rows of one dtype, got {k.dtype} and {v.dtype}")
    if k.dim() != 3 or k.shape != v.shape or tuple(k.shape[1:]) != (H, D):
        raise ValueError(f"k and v must be [T, {H}, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if v.device != k.device:
        raise ValueError(f"v is on {v.device}, not on {k.device}")
    _ints(slots, "slots", torch.int64, 1, k.device)
    if slots.shape[0] != k.shape[0]:
        raise ValueError(f"{slots.shape[0]} slots for {k.shape[0]} rows")
    k, v = _aligned_rows(k), _aligned_rows(v)
    pool = _pool_struct(k_pages, v_pages, k_scale, v_scale, 8)
    with _on(k.device):
        st = _lib.lib().hyq_paged8_append(k.data_ptr(), *_row_strides(k), v.data_ptr(), *_row_strides(v), int(k.dtype == torch.float16),
                                          slots.data_ptr(), k.shape[0], H, D, ctypes.byref(pool), _stream(k.device))
    _lib.check(st, "paged8_append")


def paged8_gather(slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows [T, H, D] of slots (int64 [T]) as bf16 (exact) or fp16:
    code * scale rounded once; zeros for slots outside the pool."""
    fx, stream = _fast(slots)
    if fx and dtype in _HALF:
        try:
            st, k, v = fx.paged8_gather(slots, k_pages, v_pages, k_scale, v_scale, dtype == torch.float16, stream)
            if st == 0:
                return k, v
        except TypeError:
            pass
    _require_gpu(slots, "slots")
    _ints(slots, "slots", torch.int64, 1, slots.device)
    N, H, P, D = _check_pool8(k_pages, v_pages, k_scale, v_scale, slots.device)
    if dtype not in _HALF:
        raise ValueError(f"paged8_gather gives bf16 or fp16 rows, not {dtype}")
    T = slots.shape[0]
    k, v = (torch.empty(T, H, D, dtype=dtype, device=slots.device) for _ in range(2))
    pool = _pool_struct(k_pages, v_pages, k_scale, v_scale, 8)
    with _on(slots.device):
        st = _lib.lib().hyq_paged8_gather(slots.data_ptr(), T, H, D, ctypes.byref(pool), int(dtype == torch.float16), k.data_ptr(),
                                          v.data_ptr(), _stream(slots.device))
    _lib.check(st, "paged8_gather")
    return k, v


def paged8_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                     block_table: torch.Tensor, seq_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                     sm_scale: Optional[float] = None, window: int = 0, return_lse: bool = False,
                     out: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """paged_attention over an 8-bit pool: causal attention of the new tokens of R
    requests over their cached tokens (their own among them: append first), the
    same arguments, masks and results.  A row that sees a key of a block whose K
    or V scale is NaN, or not within [2^-40, 2^48], is NaN."""
    return _attend("paged8_attention", 8, _check_pool8, q, k_pages, v_pages, k_scale, v_scale, block_table, seq_lens, cu_seqlens, sm_scale,
                   window, return_lse, out)
