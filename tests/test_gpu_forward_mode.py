"""The gated layer and residual_norm have no forward-mode differentiation: a tangent raises instead of being lost."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import ksmm_b200 as kb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("learns", [False, True])
@pytest.mark.parametrize("which", ["x", "factor", "bias"])
def test_gated(which, learns, native, monkeypatch):
    if not native:
        monkeypatch.setattr(kb.kernel, "_native", None)
    torch.manual_seed(0)
    layer = kb.KSGatedLinear([(6, 64, 64, 1), (1, 512, 192, 2)], dtype=torch.bfloat16, requires_grad=learns)
    x = torch.randn(40, 384, device="cuda").bfloat16()
    plain = layer(x).detach()
    with fw.dual_level():
        t = {"x": x, "factor": layer.factors[1].detach(), "bias": layer.bias.detach()}
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        factors = [layer.factors[0], t["factor"]]
        for call in (kb.kernel.gated_layer, kb.gated_chain_forward):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(t["x"], factors, layer.patterns, False, t["bias"])
        assert torch.equal(layer(x).detach(), plain)   # no tangent, no refusal


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("learns", [False, True])
@pytest.mark.parametrize("which", ["x", "y", "weight", "scale", "gate"])
def test_norm(which, learns, native, monkeypatch):
    if not native:
        monkeypatch.setattr(kb.norm, "_native", None)
    rows = lambda *s: torch.randn(*s, device="cuda")
    t = dict(x=rows(6, 64), y=rows(6, 64), weight=rows(64), scale=rows(2, 64), gate=rows(2, 64), bias=rows(64).requires_grad_(learns))
    plain = kb.residual_norm(**t)
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            kb.residual_norm(**{**t, which: fw.make_dual(t[which], torch.ones_like(t[which]))})
        for a, b in zip(kb.residual_norm(**t), plain):
            assert torch.equal(a, b)
