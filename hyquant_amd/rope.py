"""Rotation of queries and keys on MI355X, with the norms of their heads, on its
own and on the way into a paged cache.

A decoder's attention rotates the queries and keys of each head by their
position, and in some models normalises them first (Qwen3's q_norm and k_norm).
qk_norm_rope does both for all heads in one launch:

    y = x / sqrt(mean(x^2) + eps) * w                        (where there is a weight)
    (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin)

for the channel pairs (i, i + R/2), or (2i, 2i + 1) with interleaved=True, of the
first R channels; cos and sin are tables [rows, R/2] of one row per position (the
half of Hugging Face's rotary embedding: cos[..., :R // 2]).  paged_rope_append
rotates the queries, and the keys on their way into the pages of a 4-bit
(hyquant_amd.paged) or 8-bit (hyquant_amd.paged8) cache.

Arithmetic is in 32 bits and rounded once; keys that become codes have those of a
rotation in 64 bits.  Inference only: inputs that record gradients or carry
forward-mode tangents are refused.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .decode_d_stage import _HALF, _require_gpu, _stream
from .paged import _aligned_rows, _check_pool, _fast, _ints, _on, _row_strides
from .paged8 import _check_pool8, _pool_struct

_TABLE_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _differentiated(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd records a gradient of one of the tensors, or carries its tangent (forward mode, which no_grad
    does not stop), or a function transform wraps it."""
    grad = torch.is_grad_enabled()
    return any(t is not None and ((grad and t.requires_grad) or torch._C._functorch.is_functorch_wrapped_tensor(t)
                                  or forward_ad.unpack_dual(t).tangent is not None) for t in tensors)


def _no_grad(*tensors: Optional[torch.Tensor]) -> None:
    if _differentiated(*tensors):
        raise ValueError("inputs that record gradients or carry tangents are not supported: detach them, or call it under "
                         "torch.no_grad() (which forward mode ignores)")


def _rows(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in _HALF or t.dtype != like.dtype:
        raise ValueError(f"{name} must be a bf16 or fp16 tensor of q's dtype")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    if t.shape[:-2] != like.shape[:-2] or t.shape[-1] != like.shape[-1]:
        raise ValueError(f"q and {name} are of shapes {tuple(like.shape)} and {tuple(t.shape)}")


def _aligned4(t: torch.Tensor) -> torch.Tensor:
    """t [B, N, H, D] with contiguous channels and 16-byte aligned rows (a copy if it has others)."""
    strides = [s for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1]
    if t.numel() and (t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in strides)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """The strides (batch, token, head) of t [B, N, H, D]; 0 where there is one alone, whatever t says."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3]))


def _weight(w: Optional[torch.Tensor], name: str, like: torch.Tensor) -> Optional[torch.Tensor]:
    if w is None:
        return None
    if not isinstance(w, torch.Tensor) or w.dtype not in (torch.float32, like.dtype) or tuple(w.shape) != (like.shape[-1],):
        raise ValueError(f"{name} must be a tensor [{like.shape[-1]}] of fp32 or q's dtype")
    if w.device != like.device:
        raise ValueError(f"{name} is on {w.device}, not on {like.device}")
    return w if w.stride(0) == 1 and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)


def _params(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    """(the parameter block, what it points to) of rows q, k [B, N, heads, D]; the outputs are the caller's to set."""
    B, N, _, D = q.shape
    if D not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, got {D}")
    for t, name in ((cos, "cos"), (sin, "sin")):
        if not isinstance(t, torch.Tensor) or t.dtype not in _TABLE_TYPES or t.dim() not in (2, 3):
            raise ValueError(f"{name} must be an fp32, bf16 or fp16 table [rows, R / 2] or [batch, rows, R / 2]")
        if t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, not on {q.device}")
    if cos.shape != sin.shape or cos.dtype != sin.dtype:
        raise ValueError("cos and sin must be of one shape and dtype")
    half = cos.shape[-1]
    if half == 0 or half % 8 or 2 * half > D:
        raise ValueError(f"tables must have R / 2 columns, R a multiple of 16 up to the head dim {D}: got {half}")
    rows = cos.shape[-2]
    if positions is not None:
        if cos.dim() != 2:
            raise ValueError("positions need tables of two dimensions")
        if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int64 or tuple(positions.shape) not in ((B * N,), (B, N)):
            raise ValueError(f"positions must be an int64 tensor of the {B * N} tokens")
        if positions.device != q.device:
            raise ValueError(f"positions are on {positions.device}, not on {q.device}")
        positions = positions.contiguous()
        if rows == 0 and B * N:
            raise ValueError("the tables have no rows")
    elif rows < N or (cos.dim() == 3 and cos.shape[0] not in (1, B)):
        raise ValueError(f"without positions the tables need {N} rows (and a batch of 1 or {B}): got {tuple(cos.shape)}")
    strides = [s for s, n in zip(cos.stride()[:-1], cos.shape[:-1]) if n > 1]
    if (cos.stride() != sin.stride() or cos.stride(-1) != 1 or cos.data_ptr() % 16 or sin.data_ptr() % 16 or any(s % 8 for s in strides)):
        cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
    if not eps >= 0 or eps == float("inf"):
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    qw, kw = _weight(q_weight, "q_weight", q), _weight(k_weight, "k_weight", k)
    if qw is not None and kw is not None and qw.dtype != kw.dtype:
        qw, kw = qw.float(), kw.float()
    q, k = _aligned4(q), _aligned4(k)
    p = _lib.RopeParams()
    p.q, (p.q_stride_b, p.q_stride_n, p.q_stride_h) = q.data_ptr(), _strides(q)
    p.k, (p.k_stride_b, p.k_stride_n, p.k_stride_h) = k.data_ptr(), _strides(k)
    p.cos, p.sin, p.table_rows = cos.data_ptr(), sin.data_ptr(), rows
    p.table_stride_m = cos.stride(-2) if rows > 1 else 0
    p.table_stride_b = cos.stride(0) if cos.dim() == 3 and cos.shape[0] > 1 else 0
    p.positions = None if positions is None else positions.data_ptr()
    p.q_weight, p.k_weight = (None if w is None else w.data_ptr() for w in (qw, kw))
    p.eps, p.batch, p.n = eps, B, N
    p.q_heads, p.k_heads, p.head_dim, p.rotary = q.shape[2], k.shape[2], D, 2 * half
    p.interleaved, p.dtype_fp16, p.table_type = int(bool(interleaved)), int(q.dtype == torch.float16), _TABLE_TYPES[cos.dtype]
    w = qw if qw is not None else kw
    p.weight_fp32 = int(w is not None and w.dtype == torch.float32)
    return p, (q, k, cos, sin, positions, qw, kw)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor] = None,
                 *, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys rotated by their positions, normalised first where there is a weight.

    q [..., H_Q, D] and k [..., H_K, D], bf16 or fp16 of any strides, are the rows
    of T tokens ([T, heads, D]) or of a batch of sequences ([B, N, heads, D]), D 64 or
    128.  cos and sin are tables [rows, R/2] of fp32, bf16 or fp16, R a multiple of
    16 up to D: token t has row positions[t] (int64, one for each token), without
    positions the tokens of a sequence have the rows from 0 on, where tables [B or 1,
    rows, R/2] give each sequence its own.  A token whose position is outside the
    table, as the -1 of a padded batch's, has rows of zeros.  q_weight and k_weight
    [D]: RMS norm of each head, in fp32 or q's dtype.

    Returns (q, k) of the inputs' shapes and dtype, contiguous."""
    fx, stream = _fast(q)
    if fx:
        try:
            st, qo, ko = fx.qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, stream)
            if st == 0:
                return qo, ko
        except TypeError:
            pass
    _require_gpu(q, "q")
    _no_grad(q, k, cos, sin, q_weight, k_weight)
    if q.dtype not in _HALF or q.dim() not in (3, 4):
        raise ValueError(f"qk_norm_rope expects bf16 or fp16 rows [T, heads, D] or [B, N, heads, D], got {q.dtype} of {q.dim()} dimensions")
    _rows(k, "k", q)
    q4, k4 = (t if t.dim() == 4 else t.unsqueeze(0) for t in (q, k))
    p, held = _params(q4, k4, cos, sin, positions, q_weight, k_weight, eps, interleaved)
    qo, ko = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    p.q_out, p.k_out = qo.data_ptr(), ko.data_ptr()
    with _on(q.device):
        st = _lib.lib().hyq_qk_norm_rope(ctypes.byref(p), _stream(q.device))
    _lib.check(st, "qk_norm_rope")
    del held
    return qo, ko


def paged_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None,
                      k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """Rotate q, and put k, rotated, and v into their slots: one launch for what
    qk_norm_rope and paged_append (or paged8_append) do in two.

    q [T, H_Q, D], k and v [T, heads, D]; cos, sin, positions, weights, eps and
    interleaved as qk_norm_rope's; slots int64 [T].  The pool's scales say what it is: fp16
    [pages, heads, page] a cache of 4 bits (paged_append), fp32 [pages, heads, page / 16] one
    of 8 (paged8_append, whose contract of slots holds here too).  The codes are those
    of the rotated keys before any rounding to 16 bits.  A token whose position is
    outside the table or whose slot is outside the pool writes nothing; q's rows
    are zero where the position is.  Returns q rotated, contiguous."""
    fx, stream = _fast(q)
    if fx:
        try:
            st, qo = fx.rope_append(q, k, v, cos, sin, positions, slots, k_pages, v_pages, k_scale, v_scale, q_weight, k_weight, eps,
                                    interleaved, stream)
            if st == 0:
                return qo
        except TypeError:
            pass
    _require_gpu(q, "q")
    _no_grad(q, k, v, cos, sin, q_weight, k_weight)
    if q.dtype not in _HALF or q.dim() != 3:
        raise ValueError(f"paged_rope_append expects bf16 or fp16 rows [T, heads, D], got {q.dtype} of {q.dim()} dimensions")
    _rows(k, "k", q)
    _rows(v, "v", q)
    eight = isinstance(k_scale, torch.Tensor) and k_scale.dtype == torch.float32
    N, H, P, D = (_check_pool8 if eight else _check_pool)(k_pages, v_pages, k_scale, v_scale, q.device)
    T = q.shape[0]
    if tuple(k.shape[1:]) != (H, D) or k.shape != v.shape:
        raise ValueError(f"k and v must be [{T}, {H}, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    _ints(positions, "positions", torch.int64, 1, q.device)
    _ints(slots, "slots", torch.int64, 1, q.device)
    if slots.shape[0] != T:
        raise ValueError(f"{slots.shape[0]} slots for {T} rows")
    p, held = _params(q.unsqueeze(0), k.unsqueeze(0), cos, sin, positions, q_weight, k_weight, eps, interleaved)
    v = _aligned_rows(v)
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    p.q_out = qo.data_ptr()
    pool = _pool_struct(k_pages, v_pages, k_scale, v_scale, 8 if eight else 4)
    with _on(q.device):
        st = _lib.lib().hyq_paged_rope_append(ctypes.byref(p), v.data_ptr(), *_row_strides(v), slots.data_ptr(), ctypes.byref(pool),
                                              _stream(q.device))
    _lib.check(st, "paged_rope_append")
    del held
    return qo
