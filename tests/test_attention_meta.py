"""KSAttention built on the meta device, and what changes of type and device leave of its rotation; no GPU."""
import torch

import ksmm_b200 as kb

Q = [(6, 64, 64, 1), (1, 192, 192, 2)]


def layer(**kw):
    return kb.KSAttention(Q, Q, 6, device="meta", **kw)


def test_frequencies_of_a_layer_from_meta():
    for dtype in (torch.float32, torch.bfloat16):
        attn = layer(dtype=dtype, rotary_base=500.0, rotary_dim=48)
        assert attn.frequencies.is_meta and attn.frequencies.dtype == torch.float64
        attn.half()
        assert attn.frequencies.is_meta and attn.frequencies.dtype == torch.float64
        attn.to_empty(device="cpu")
        assert torch.equal(attn.frequencies, kb.rotary_frequencies(24, 500.0, "cpu"))
        assert "frequencies" not in attn.state_dict()
    assert layer(rotary_base=None).to_empty(device="cpu").frequencies is None
    assert layer(rotary_dim=0).to_empty(device="cpu").frequencies.shape == (0,)


def test_frequencies_stay():
    attn = layer().to_empty(device="cpu")
    attn.frequencies.mul_(0.125)  # (positions of a longer context)
    want = attn.frequencies.clone()
    for change in (lambda a: a.half(), lambda a: a.float(), lambda a: a.to(torch.bfloat16), lambda a: a.to_empty(device="cpu"),
                   lambda a: a.to("cpu"), lambda a: a.double()):
        change(attn)
        assert attn.frequencies.dtype == torch.float64 and torch.equal(attn.frequencies, want)
