"""Refusals of the rotation and of the 8-bit pages that need no GPU: the C ABI
rejects bad arguments on the host before any launch, and the Python layer's
checks."""

import ctypes
import os

import pytest
import torch


def _L():
    from hyquant_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libhyq.so not built")
    return _lib, _lib.lib()


def _params(_lib, **kw):
    p = _lib.RopeParams()
    p.q, p.q_stride_b, p.q_stride_n, p.q_stride_h, p.q_out = 256, 0, 4096, 128, 512
    p.k, p.k_stride_b, p.k_stride_n, p.k_stride_h, p.k_out = 256, 0, 1024, 128, 512
    p.cos, p.sin, p.table_stride_m, p.table_rows, p.positions = 256, 256, 64, 100, 256
    p.eps, p.batch, p.n, p.q_heads, p.k_heads, p.head_dim, p.rotary = 1e-6, 1, 5, 32, 8, 128, 128
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _pool(_lib, bits, **kw):
    p = _lib.PagedPool(4096, 8192, 32768, 4096, 4096, 8192, 512, 64, 100, 64, bits)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _bad_params(E, N):
    return ((dict(head_dim=96), N), (dict(batch=-1), E), (dict(n=-1), E), (dict(q_heads=-1), E), (dict(k_heads=70000), N),
            (dict(dtype_fp16=2), E), (dict(rotary=24), N), (dict(rotary=144), N), (dict(table_type=3), E), (dict(weight_fp32=2), E),
            (dict(interleaved=2), E), (dict(eps=float("nan")), E), (dict(eps=-1.0), E), (dict(eps=float("inf")), E), (dict(n=1 << 40), N),
            (dict(n=1 << 26), N), (dict(q=None), E), (dict(q_out=None), E), (dict(k=None), E), (dict(q=264), E),
            (dict(q_stride_n=100), E), (dict(k_stride_h=4), E), (dict(q_out=8), E), (dict(q_weight=8), E), (dict(positions=4), E),
            (dict(table_rows=-1), E), (dict(table_rows=0), E), (dict(positions=None, table_rows=4), E), (dict(cos=None), E),
            (dict(sin=8), E), (dict(table_stride_m=4), E))


def test_rotation_host_validation():
    _lib, L = _L()
    E, N = _lib.HYQ_EINVAL, _lib.HYQ_ENOTSUP
    for bad, code in _bad_params(E, N) + ((dict(k_out=None), E), (dict(batch=1 << 20, n=1 << 20), N), (dict(batch=1 << 62, n=2), N)):
        assert L.hyq_qk_norm_rope(_params(_lib, **bad), None) == code, bad
    assert L.hyq_qk_norm_rope(None, None) == E
    for none in (dict(batch=0), dict(n=0), dict(q_heads=0, k_heads=0)):
        assert L.hyq_qk_norm_rope(_params(_lib, **none), None) == _lib.HYQ_OK


@pytest.mark.parametrize("bits", [4, 8])
def test_rotated_append_host_validation(bits):
    _lib, L = _L()
    E, N = _lib.HYQ_EINVAL, _lib.HYQ_ENOTSUP
    call = lambda p, pool, v=256, vt=1024, vh=128, slots=256: L.hyq_paged_rope_append(p, v, vt, vh, slots, pool, None)  # noqa: E731
    for bad, code in _bad_params(E, N) + ((dict(batch=2), E), (dict(k_heads=0), E)):
        assert call(_params(_lib, **bad), _pool(_lib, bits)) == code, bad
    for bad, code in ((dict(page_size=48), N), (dict(page_size=8), N), (dict(num_pages=-1), E), (dict(k_pages=None), E), (dict(v_pages=8), E),
                      (dict(p_stride_head=8), E), (dict(k_scale=4097), E), (dict(v_scale=None), E)):
        assert call(_params(_lib), _pool(_lib, bits, **bad)) == code, bad
    assert call(_params(_lib), None) == E and call(_params(_lib), _pool(_lib, 6)) == E
    for bad in (dict(v=None), dict(v=264), dict(vt=100), dict(slots=None), dict(slots=260)):
        assert call(_params(_lib), _pool(_lib, bits), **bad) == E, bad
    assert call(_params(_lib, n=0), _pool(_lib, bits), v=None, slots=None) == _lib.HYQ_OK


def test_append8_and_gather8_host_validation():
    _lib, L = _L()
    E, N = _lib.HYQ_EINVAL, _lib.HYQ_ENOTSUP
    ok = [256, 1024, 128, 256, 1024, 128, 0, 256, 5, 8, 128, _pool(_lib, 8), None]
    for at, value, code in ((0, None, E), (0, 264, E), (1, 1020, E), (6, 2, E), (7, None, E), (8, -1, E), (9, 0, E), (10, 100, N),
                            (8, 1 << 28, N), (11, None, E), (11, _pool(_lib, 4), E), (11, _pool(_lib, 8, page_size=20), N),
                            (11, _pool(_lib, 8, k_scale=4098), E)):
        args = list(ok)
        args[at] = value
        assert L.hyq_paged8_append(*args) == code, (at, value)
    args = list(ok)
    args[8] = 0
    assert L.hyq_paged8_append(*args) == _lib.HYQ_OK
    ok = [256, 5, 8, 128, _pool(_lib, 8), 0, 256, 256, None]
    for at, value, code in ((0, None, E), (1, -1, E), (2, 0, E), (3, 32, N), (4, _pool(_lib, 4), E), (5, 2, E), (6, None, E), (7, 264, E),
                            (1, 1 << 28, N)):
        args = list(ok)
        args[at] = value
        assert L.hyq_paged8_gather(*args) == code, (at, value)


def test_structs_are_the_headers():
    """The ctypes mirrors have the C compiler's layout (all fields naturally aligned, none padded)."""
    from hyquant_amd import _lib
    for S in (_lib.RopeParams, _lib.PagedPool):
        assert ctypes.sizeof(S) == sum(ctypes.sizeof(t) for _, t in S._fields_) and ctypes.sizeof(S) % 8 == 0


def test_python_checks():
    import hyquant_amd as hq
    from hyquant_amd import paged8, rope
    x = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    cos = torch.zeros(5, 32)
    good = (x, x, cos, cos, None, None, None, 1e-6, False)
    assert rope._params(*good)[0].rotary == 64
    w = torch.zeros(64)
    for at, value, word in ((0, x[..., :32], "head dim"), (2, cos[0], "cos"), (2, cos.double(), "cos"), (3, cos[:4], "one shape"),
                            (3, cos.half(), "one shape"), (4, torch.zeros(5, dtype=torch.int64), "positions"),
                            (4, torch.zeros(6, dtype=torch.int32), "positions"), (5, w[:32], "q_weight"), (6, w.double(), "k_weight"),
                            (5, w.half(), "q_weight"), (7, -1.0, "eps"), (7, float("nan"), "eps")):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=word):
            rope._params(*args)
    for c in (cos[:, :12], torch.zeros(5, 40), torch.zeros(5, 0), cos[:2], torch.zeros(3, 5, 32)):
        with pytest.raises(ValueError, match="tables"):
            rope._params(x, x, c, c, None, None, None, 1e-6, False)
    with pytest.raises(ValueError, match="two dimensions"):
        c = torch.zeros(2, 5, 32)
        rope._params(x, x, c, c, torch.zeros(6, dtype=torch.int64), None, None, 1e-6, False)
    # weights of two dtypes both become fp32; strides of a dimension of one do not count
    p, held = rope._params(x, x, cos, cos, None, w, w.bfloat16(), 1e-6, False)
    assert p.weight_fp32 == 1 and held[-1].dtype == torch.float32
    odd = torch.zeros(1, 3, 1, 68, dtype=torch.bfloat16)[..., :64]
    assert rope._aligned4(odd) is not odd and rope._aligned4(odd[:, :1]).data_ptr() == odd.data_ptr()
    with pytest.raises(ValueError, match="GPU"):
        hq.qk_norm_rope(x, x, cos, cos)
    pool = tuple(torch.zeros(3, 2, 32, 64, dtype=torch.int8) for _ in range(2)) + tuple(torch.zeros(3, 2, 2) for _ in range(2))
    cpu = torch.device("cpu")
    assert paged8._check_pool8(*pool, cpu) == (3, 2, 32, 64)
    kp, vp, ks, vs = pool
    for args, word in (((kp.short(), vp, ks, vs), "k_pages"), ((kp, vp, ks.half(), vs), "k_scale"), ((kp, vp, ks[..., :1], vs), "shapes"),
                       ((kp, vp[:2], ks, vs), "shapes"), ((kp[:, :, :24], vp[:, :, :24], ks, vs), "page size"),
                       ((kp[..., :48], vp[..., :48], ks, vs), "head dim"),
                       ((kp.transpose(0, 1).contiguous().transpose(0, 1), vp, ks, vs), "strides")):
        with pytest.raises(ValueError, match=word):
            paged8._check_pool8(*args, cpu)
    for call in (lambda: hq.paged8_append(x[0], x[0], torch.zeros(3, dtype=torch.int64), *pool),
                 lambda: hq.paged8_gather(torch.zeros(3, dtype=torch.int64), *pool)):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("family", ["llama", "qwen"])
def test_fused_rope_on_the_cpu_is_the_models_own(family):
    transformers = pytest.importorskip("transformers")
    from hyquant_amd.patch import patch_attention_forward_model
    torch.manual_seed(0)
    common = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                  vocab_size=128, max_position_embeddings=512, attn_implementation="sdpa")
    make = (lambda: transformers.LlamaForCausalLM(transformers.LlamaConfig(**common))) if family == "llama" else (
        lambda: transformers.Qwen3ForCausalLM(transformers.Qwen3Config(**common)))
    ref, pat = make().eval(), make().eval()
    pat.load_state_dict(ref.state_dict())
    patch_attention_forward_model(pat, mode="dense", fused_rope=True)
    ids = torch.randint(0, 128, (1, 40), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        assert torch.equal(ref(ids).logits, pat(ids).logits)
