"""Forward-mode derivatives: the rotation refuses inputs that carry tangents, and a
patched model with fused_rope takes its own operations for them."""

import pytest
import torch
from torch.autograd import forward_ad

import hyquant_amd as hq
from tests import rope_util as U
from tests.test_gpu_patch import W, _model
from tests.test_gpu_rope import BF, DEV, FL, as_long, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_tangents_are_refused(native, monkeypatch):
    from hyquant_amd import decode_d_stage as dd
    if not native:
        monkeypatch.setattr(dd, "_FX", False)
    g = gen(0)
    cos, sin = U.tables(4, 64, device=DEV)
    x, w = randn(g, 2, 2, 64), randn(g, 64, dtype=FL)
    pool = U.pool8(g, 1, 2, 16, 64, DEV)
    before = [t.clone() for t in pool]
    at = as_long([0, 1])
    args = dict(q=x, k=x, cos=cos, sin=sin, q_weight=w, k_weight=w)
    want = hq.qk_norm_rope(**args)
    with forward_ad.dual_level():
        for name, t in args.items():
            dual = dict(args, **{name: forward_ad.make_dual(t, torch.ones_like(t))})
            with pytest.raises(ValueError, match="tangents"):
                hq.qk_norm_rope(**dual)
            with torch.no_grad(), pytest.raises(ValueError, match="tangents"):
                hq.qk_norm_rope(**dual)
            with pytest.raises(ValueError, match="tangents"):
                hq.paged_rope_append(**dual, v=x, positions=at, slots=at, k_pages=pool[0], v_pages=pool[1], k_scale=pool[2], v_scale=pool[3])
        v = forward_ad.make_dual(x, x)
        with pytest.raises(ValueError, match="tangents"):
            hq.paged_rope_append(x, x, v, cos, sin, at, at, *pool)
        assert all(torch.equal(a, b) for a, b in zip(hq.qk_norm_rope(**args), want))
        with torch.inference_mode():         # (torch's own operations carry none here either)
            assert all(torch.equal(a, b) for a, b in zip(hq.qk_norm_rope(v, **{n: t for n, t in args.items() if n != "q"}), want))
    assert all(torch.equal(a, b) for a, b in zip(pool, before))


@pytest.mark.parametrize("native", [True, False])
def test_function_transforms_are_refused(native, monkeypatch):
    from hyquant_amd import decode_d_stage as dd
    if not native:
        monkeypatch.setattr(dd, "_FX", False)
    cos, sin = U.tables(4, 64, device=DEV)
    x = randn(gen(1), 3, 2, 2, 64)
    for transformed in (lambda: torch.func.vmap(lambda q: hq.qk_norm_rope(q, q, cos, sin)[0])(x),
                        lambda: torch.func.jvp(lambda q: hq.qk_norm_rope(q, q, cos, sin)[0], (x[0],), (x[1],)),
                        lambda: torch.func.grad(lambda q: hq.qk_norm_rope(q, q, cos, sin)[0].float().sum())(x[0])):
        with pytest.raises(ValueError, match="not supported"):
            transformed()


@pytest.mark.parametrize("family", ["llama", "qwen"])
@pytest.mark.parametrize("no_grad", [False, True])
def test_a_patched_model_carries_tangents(family, no_grad):
    from hyquant_amd import patch
    m = _model(family).requires_grad_(False)
    at = m.model.layers[0].self_attn
    g = gen(4)
    x, t = (randn(g, 2, 19, m.config.hidden_size) for _ in range(2))
    cos, sin = m.model.rotary_emb(x, torch.arange(19, device=DEV)[None])
    outs = []
    for fused in (False, True):
        fwd = patch.build_attention_forward(family, mode="dense", window_size=W, top_ratio=0.05, fused_rope=fused)
        with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
            out = forward_ad.unpack_dual(fwd(at, forward_ad.make_dual(x, t), (cos, sin))[0])
            outs.append((out.primal.clone(), out.tangent.clone()))
        outs[-1] += torch.func.jvp(lambda y: fwd(at, y, (cos, sin))[0], (x,), (t,))
    for a, b in zip(*outs):
        assert a.dtype == BF and torch.equal(a, b)
    assert bool((outs[1][1] != 0).any())
