"""The paged operators' refusals that need no GPU: the C ABI rejects bad
arguments on the host before any launch, and the Python layer's shape checks."""

import os

import pytest
import torch


def _L():
    from hyquant_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libhyq.so not built")
    return _lib, _lib.lib()


def _params(_lib, **kw):
    p = _lib.PagedParams()
    p.q, p.q_stride_t, p.q_stride_h, p.out, p.o_stride_t, p.o_stride_h = 256, 4096, 128, 512, 4096, 128
    p.k_pages, p.v_pages, p.p_stride_page, p.p_stride_head = 4096, 8192, 8 * 64 * 64, 64 * 64
    p.k_scale, p.v_scale, p.s_stride_page, p.s_stride_head = 4096, 8192, 8 * 64, 64
    p.block_table, p.bt_stride, p.seq_lens, p.num_pages, p.page_size, p.max_pages = 256, 16, 256, 100, 64, 16
    p.num_requests, p.num_tokens, p.kv_heads, p.kv_repeat, p.head_dim, p.sm_scale = 4, 4, 8, 4, 128, 0.1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_attention_host_validation():
    _lib, L = _L()
    assert L.hyq_paged_attention_workspace_size(_params(_lib)) > 0
    E, N = _lib.HYQ_EINVAL, _lib.HYQ_ENOTSUP
    for bad, code in ((dict(head_dim=96), N), (dict(page_size=48), N), (dict(page_size=8), N), (dict(page_size=512), N),
                      (dict(kv_repeat=0), N), (dict(kv_heads=0), E), (dict(num_pages=-1), E), (dict(window=-1), E),
                      (dict(num_tokens=-1), E), (dict(num_tokens=5), E), (dict(q=None), E), (dict(q=260), E),
                      (dict(q_stride_h=100), E), (dict(out=4), E), (dict(o_stride_t=2), E), (dict(seq_lens=None), E),
                      (dict(block_table=None), E), (dict(k_pages=None), E), (dict(k_pages=8), E), (dict(p_stride_head=8), E),
                      (dict(dtype_fp16=2), E), (dict(zero_tail=4), E), (dict(sm_scale=float("nan")), E),
                      (dict(max_pages=1 << 25), N), (dict(num_tokens=1 << 29, cu_seqlens=256), N)):
        p = _params(_lib, **bad)
        assert L.hyq_paged_attention_workspace_size(p) == 0, bad
        assert L.hyq_paged_attention(p, 4096, 1 << 40, None) == code, bad
    assert L.hyq_paged_attention(_params(_lib), 4096, 16, None) == _lib.HYQ_ENOSPC
    assert b"workspace" in L.hyq_last_error()
    assert L.hyq_paged_attention(_params(_lib), 4100, 1 << 40, None) == E
    assert L.hyq_paged_attention(_params(_lib, num_requests=0, num_tokens=0), None, 0, None) == _lib.HYQ_OK
    assert L.hyq_paged_attention(None, None, 0, None) == E


def test_workspace_does_not_grow_with_the_lengths():
    """Partial results are kept for the split tiles alone: a long prompt's or a
    large batch's workspace is its schedule."""
    _lib, L = _L()
    small = L.hyq_paged_attention_workspace_size(_params(_lib))
    many = L.hyq_paged_attention_workspace_size(_params(_lib, num_requests=4096, num_tokens=4096))
    long = L.hyq_paged_attention_workspace_size(_params(_lib, num_requests=1, num_tokens=1 << 17, cu_seqlens=256))
    assert small < 64 << 20 and many < 256 << 20 and long < 256 << 20


def test_batch_host_validation():
    _lib, L = _L()
    E, N = _lib.HYQ_EINVAL, _lib.HYQ_ENOTSUP
    ok = [256, 256, 2, 256, 4, 4, 256, 8, 16, 6, 256, 256, 256, 256, 256, None]
    for at, value, code in ((0, None, E), (1, 258, E), (2, -1, E), (2, 16385, N), (3, None, E), (6, None, E), (8, 17, N),
                            (9, -1, E), (10, None, E), (12, 260, E), (13, None, E), (14, None, E)):
        args = list(ok)
        args[at] = value
        assert L.hyq_paged_batch(*args) == code, (at, value)


def test_append_and_gather_host_validation():
    _lib, L = _L()
    E, N = _lib.HYQ_EINVAL, _lib.HYQ_ENOTSUP
    ok = [256, 1024, 128, 256, 1024, 128, 0, 256, 5, 8, 128, 4096, 4096, 32768, 4096, 4096, 4096, 512, 64, 100, 64, None]
    for at, value, code in ((0, None, E), (0, 264, E), (1, 1020, E), (6, 2, E), (7, None, E), (8, -1, E), (9, 0, E), (10, 100, N),
                            (11, None, E), (13, 8, E), (15, 4097, E), (19, -1, E), (20, 40, N), (8, 1 << 28, N)):
        args = list(ok)
        args[at] = value
        assert L.hyq_paged_append(*args) == code, (at, value)
    args = list(ok)
    args[8] = 0
    assert L.hyq_paged_append(*args) == _lib.HYQ_OK
    ok = [256, 5, 8, 128, 4096, 4096, 32768, 4096, 4096, 4096, 512, 64, 100, 64, 0, 256, 256, None]
    for at, value, code in ((0, None, E), (1, -1, E), (3, 32, N), (13, 40, N), (14, 2, E), (15, None, E), (16, 264, E), (5, None, E)):
        args = list(ok)
        args[at] = value
        assert L.hyq_paged_gather(*args) == code, (at, value)


def test_pool_checks():
    from hyquant_amd import paged
    from tests.paged_util import make_pool
    pool = make_pool(torch.Generator().manual_seed(0), 3, 2, 16, 64, "cpu")
    cpu = torch.device("cpu")
    assert paged._check_pool(*pool, cpu) == (3, 2, 16, 64)
    kp, vp, ks, vs = pool
    for args, word in (((kp.short(), vp, ks, vs), "k_pages"), ((kp, vp[0], ks, vs), "v_pages"), ((kp, vp, ks[:2], vs), "shapes"),
                       ((kp[:, :, :15], vp[:, :, :15], ks[:, :, :15], vs[:, :, :15]), "page size"),
                       ((kp[..., :24], vp[..., :24], ks, vs), "head dim"),
                       ((kp.flip(0).transpose(2, 3).contiguous().transpose(2, 3), vp, ks, vs), "strides")):
        with pytest.raises(ValueError, match=word):
            paged._check_pool(*args, cpu)
    wide = torch.zeros(3, 2, 16, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="contiguous"):
        paged._check_pool(wide[..., :32], wide[..., 32:], ks, vs, cpu)
    with pytest.raises(ValueError, match="GPU"):
        paged.paged_attention(torch.zeros(1, 2, 64, dtype=torch.bfloat16), *pool, torch.zeros(1, 1, dtype=torch.int32),
                              torch.ones(1, dtype=torch.int32))


def test_attention_limits_of_heads_and_counters():
    _lib, L = _L()
    assert L.hyq_paged_attention_workspace_size(_params(_lib, kv_heads=1024)) > 0
    for bad, code in ((dict(kv_heads=1025), _lib.HYQ_ENOTSUP), (dict(counters=4097), _lib.HYQ_EINVAL)):
        assert L.hyq_paged_attention_workspace_size(_params(_lib, **bad)) == 0, bad
        assert L.hyq_paged_attention(_params(_lib, **bad), 4096, 1 << 40, None) == code, bad
