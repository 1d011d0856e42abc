"""GPU: when the MLP block packs its activations."""
import pytest
import torch

from vision_longformer_amd import msvit

pytestmark = pytest.mark.gpu


def test_only_a_block_that_needs_a_gradient_packs(monkeypatch):
    """a frozen block of a frozen input runs as in evaluation; one tensor that wants a gradient is enough for the 8-bit form"""
    calls = []
    real = msvit.vil_mlp_act8
    monkeypatch.setattr(msvit, "vil_mlp_act8", lambda *a: calls.append(1) or real(*a))
    mlp = msvit.Mlp(64, 256, act8=True).cuda().to(torch.bfloat16)
    x = torch.randn(50, 64, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        want = mlp(x)
    mlp.requires_grad_(False)
    assert torch.equal(mlp(x), want) and not calls
    for leaf in (x, *mlp.parameters()):
        leaf.requires_grad_(True)
        del calls[:]
        y = mlp(x)
        g, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert calls and g.shape == leaf.shape and bool(torch.isfinite(g).all())
        leaf.requires_grad_(False)
