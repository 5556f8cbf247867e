"""Patched models with fused_rope whose head norms do more than their formula: hooks,
replaced forwards, weights that a hook brings in; the modules' own calls are made then."""

import types

import pytest
import torch

from tests.test_gpu_patch import W, _model
from tests.test_gpu_rope import BF, DEV, gen, randn

pytestmark = pytest.mark.gpu


class Keys:
    """A cache that keeps the keys it is handed."""

    def update(self, k, v, layer, kw):
        self.k = k.clone()
        return k, v


def both(m, x, family="qwen", mode="dense"):
    """(output, keys) of a module's patched forward without and with fused_rope."""
    from hyquant_amd import patch
    at = m.model.layers[0].self_attn
    cos, sin = m.model.rotary_emb(x, torch.arange(x.shape[1], device=DEV)[None])
    outs = []
    for fused in (False, True):
        keys = Keys()
        fwd = patch.build_attention_forward(family, mode=mode, window_size=W, top_ratio=0.05, fused_rope=fused)
        with torch.no_grad():
            outs.append((fwd(at, x, (cos, sin), past_key_values=keys)[0], keys.k))
    return outs


def same(outs):
    return all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(*outs))


def model():
    m = _model("qwen")
    g = gen(2)
    for n in (m.model.layers[0].self_attn.q_norm, m.model.layers[0].self_attn.k_norm):
        n.weight.data.copy_(1 + 0.3 * torch.randn(n.weight.shape, generator=g))
    return m, randn(g, 1, 23, m.config.hidden_size)


def test_plain_norms_are_fused():
    """(So that the tests below show something: the two ways round differently.)"""
    m, x = model()
    assert not same(both(m, x))


@pytest.mark.parametrize("kind", ["forward", "pre", "global", "method"])
@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
def test_hooks_and_replaced_forwards_run(kind, which):
    m, x = model()
    norm = getattr(m.model.layers[0].self_attn, which)
    plain = both(m, x)[0]
    calls = []

    def hook(mod, args, out=None):
        if mod is norm:
            calls.append(1)
            return 2 * out if kind != "pre" else (args[0] + 1,)

    if kind == "method":
        own = norm.forward
        norm.forward = types.MethodType(lambda self, y: calls.append(1) or 2 * own(y), norm)
        handle = None
    else:
        handle = {"forward": norm.register_forward_hook, "pre": norm.register_forward_pre_hook,
                  "global": torch.nn.modules.module.register_module_forward_hook}[kind](hook)
    try:
        outs = both(m, x)
    finally:
        if handle is not None:
            handle.remove()
    assert len(calls) == 2 and same(outs)
    assert not torch.equal(outs[1][0], plain[0])


def test_weights_that_a_hook_brings_in():
    m, x = model()
    at = m.model.layers[0].self_attn
    want = both(m, x)[0]
    for n in (at.q_norm, at.k_norm):
        n.weight.data = n.weight.data.cpu()

        def bring(mod, args):
            mod.weight.data = mod.weight.data.to(DEV)

        def away(mod, args, out):
            mod.weight.data = mod.weight.data.cpu()

        n.register_forward_pre_hook(bring)
        n.register_forward_hook(away)
    outs = both(m, x)
    assert same(outs) and all(torch.equal(a, b) for a, b in zip(outs[1], want))
    assert at.q_norm.weight.device.type == "cpu"


def test_norms_of_another_class():
    m, x = model()
    at = m.model.layers[0].self_attn

    class Shifted(type(at.k_norm)):
        def forward(self, y):
            return super().forward(y) + 1

    k = Shifted(128).to(DEV, BF)
    k.load_state_dict(at.k_norm.state_dict())
    at.k_norm = k
    assert same(both(m, x))


@pytest.mark.parametrize("what", ["weights in fp16", "weights in fp64", "one weight in fp64", "keys in fp32", "angles in fp64"])
def test_types_that_the_rotation_does_not_take(what):
    """What the modules compute without fused_rope, they compute with it."""
    from hyquant_amd import patch
    m, x = model()
    at = m.model.layers[0].self_attn
    if what == "keys in fp32":
        at.k_proj.float()
        project = at.k_proj.forward
        at.k_proj.forward = lambda y: project(y.float())
    elif what != "angles in fp64":
        to = torch.float16 if "fp16" in what else torch.float64
        for n in (at.k_norm,) if "one" in what else (at.q_norm, at.k_norm):
            n.weight.data = n.weight.data.to(to)
    cos, sin = m.model.rotary_emb(x, torch.arange(x.shape[1], device=DEV)[None])
    if what == "angles in fp64":
        cos, sin = cos.double(), sin.double()
    keys = []

    class Done(Exception):
        pass

    class Only:
        def update(self, k, v, layer, kw):
            keys.append(k)
            raise Done                   # (the attention behind would want one type of all)

    for fused in (False, True):
        fwd = patch.build_attention_forward("qwen", mode="dense", window_size=W, top_ratio=0.05, fused_rope=fused)
        with torch.no_grad(), pytest.raises(Done):
            fwd(at, x, (cos, sin), past_key_values=Only())
    assert keys[0].dtype == keys[1].dtype and torch.equal(*keys)


@pytest.mark.parametrize("eps", [(1e-6, 0.5), (0.25, 1e-6), (0.5, 0.5)])
def test_each_norm_has_its_own_eps(eps):
    m, x = model()
    at = m.model.layers[0].self_attn
    at.q_norm.variance_epsilon, at.k_norm.variance_epsilon = eps
    outs = both(m, x)
    if eps[0] != eps[1]:
        assert same(outs)
    else:                                # (one launch for both; its roundings are others)
        own, fused = outs
        plain = both(model()[0], x)[0]
        far = (own[1].double() - plain[1].double()).norm()
        assert not same(outs) and (own[1].double() - fused[1].double()).norm() < far / 8
