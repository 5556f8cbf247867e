"""Patched models with fused_rope: the attention modules' own queries and keys
rotated by qk_norm_rope against 64 bits, through prompts and decode steps, and the
module's own operations where a gradient is recorded."""

import pytest
import torch

from tests import rope_util as R
from tests.test_gpu_patch import W, _ids, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("family", ["llama", "qwen"])
@pytest.mark.parametrize("mode", ["dense", "hybrid_full"])
def test_patched_models_rotate_in_one_launch(family, mode, monkeypatch):
    from hyquant_amd import patch
    m = patch.patch_attention_forward_model(_model(family), mode=mode, window_size=W, fused_rope=True)
    if family == "qwen":                 # norm weights away from one
        for i, layer in enumerate(m.model.layers):
            g = torch.Generator().manual_seed(i)
            for n in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                n.weight.data.copy_(1 + 0.3 * torch.randn(n.weight.shape, generator=g))
    seen = []

    def checked(q, k, cos, sin, **kw):
        out = fused(q, k, cos, sin, **kw)
        for x, y, w in zip((q, k), out, (kw.get("q_weight"), kw.get("k_weight"))):
            assert (w is not None) == (family == "qwen") and y.shape == x.shape and not y.requires_grad
            ref, big = R.turn(x, cos, sin, w, kw.get("eps", 1e-6))
            assert bool(((y.double() - ref).abs() <= R.tolerance(ref, big, x.dtype)).all())
        seen.append(q.shape[1])
        return out

    fused = patch.qk_norm_rope
    monkeypatch.setattr(patch, "qk_norm_rope", checked)
    cache = patch.create_cache_for_mode(mode, m.config.num_hidden_layers, window_size=W)
    n = 300
    with torch.no_grad():
        out = m.generate(_ids(n=n), max_new_tokens=4, do_sample=False, **({"past_key_values": cache} if cache is not None else {}))
    assert out.shape == (1, n + 4)
    assert seen == [n] * 2 + [1] * 6     # two layers: the prompt, then three steps


@pytest.mark.parametrize("family", ["llama", "qwen"])
def test_fused_and_own_operations_agree_as_their_roundings_do(family):
    """One attention module's queries and keys: the module's operations round up to
    five times (norm, weight, two products, sum) to bf16, the launch once, so that
    they are within six half steps of the magnitudes."""
    from hyquant_amd import patch
    m = _model(family)
    at = m.model.layers[0].self_attn
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 37, m.config.hidden_size, generator=g).to(device="cuda", dtype=torch.bfloat16)
    cos, sin = m.model.rotary_emb(x, torch.arange(37, device="cuda")[None])
    got = {}

    class Cache:
        def update(self, k, v, layer, kw):
            got.setdefault("k", []).append(k)
            return k, v

    for fused in (False, True):
        fwd = patch.build_attention_forward(family, mode="full_attention", window_size=W, top_ratio=0.05, fused_rope=fused)
        with torch.no_grad():
            fwd(at, x, (cos, sin), past_key_values=Cache())
    a, b = (t.double() for t in got["k"])
    k = at.k_proj(x).view(2, 37, -1, 128)
    _, big = R.turn(k, cos[..., :64], sin[..., :64], at.k_norm.weight if family == "qwen" else None, 1e-6)
    assert bool(((a - b).abs() <= 6 * 2.0 ** -8 * big.transpose(1, 2)).all()) and not torch.equal(a, b)


@pytest.mark.parametrize("family,frozen", [("llama", False), ("qwen", False), ("qwen", True)])
def test_gradients_take_the_modules_own_operations(family, frozen, monkeypatch):
    from hyquant_amd import patch

    def never(*a, **kw):
        raise AssertionError("called")

    monkeypatch.setattr(patch, "qk_norm_rope", never)
    ids = _ids(n=20)
    grads = []
    for fused in (False, True):
        m = patch.patch_attention_forward_model(_model(family), mode="dense", window_size=W, fused_rope=fused)
        if frozen:                       # the head norms alone are trained, in the first layer: q and k record no gradient before them
            for n, p in m.named_parameters():
                p.requires_grad_("layers.0.self_attn" in n and "_norm" in n)
        m(ids).logits.float().square().mean().backward()
        grads.append([p.grad.clone() for p in m.parameters() if p.requires_grad])
    assert len(grads[0]) >= 2 and all(torch.equal(a, b) for a, b in zip(*grads))
